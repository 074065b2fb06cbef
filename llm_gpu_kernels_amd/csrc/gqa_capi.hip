// C ABI of the segmented-KV GQA attention (include/gqa_mi355x.h).
//
// Validation mirrors _validate_attention_input / _validate_output of the
// reference (attention_cuda_compact.py:97-121): bf16, [L, heads, 128] with
// inner strides (128, 1), token stride >= heads*128 and a multiple of 8,
// 16-byte aligned bases; the current segment's length equals T.
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include <new>

#include "../../include/gqa_mi355x.h"
#include "gqa_internal.h"

namespace moe {
int capi_fail(int code, const char *fmt, ...);  // moe_capi.hip (thread-local message)
}

struct gqa_packed_plan {
  moe::GqaPackedArgs a;
  int device, cus;
};

struct gqa_paged_plan {
  moe::GqaPagedArgs a;
  int device, cus;
};

struct gqa_seg_plan {
  moe::GqaArgs a;
  moe::GqaShape shape;
  int device;
};

namespace {

constexpr int64_t kMaxTokenStride = 1LL << 25;
static_assert(63 * 2 * kMaxTokenStride + 256 < 1LL << 32, "a 64-row stage of the long-chunk kernel");

bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

int validate(const gqa_seg_desc *d, int num_cus, moe::GqaShape *shape) {
  using moe::capi_fail;
  if (!d) return capi_fail(MOE_EINVAL, "null descriptor");
  if (d->D != 128) return capi_fail(MOE_EINVAL, "head_dim must be 128 (got %d)", d->D);
  if (d->T < 0) return capi_fail(MOE_EINVAL, "T must be >= 0");
  if (d->Hkv < 1 || d->Hq < 1 || d->Hq % d->Hkv)
    return capi_fail(MOE_EINVAL, "Hq must be a positive multiple of Hkv");
  const int G = d->Hq / d->Hkv;
  if (G != 1 && G != 2 && G != 4 && G != 8)
    return capi_fail(MOE_EINVAL, "Hq / Hkv must be 1, 2, 4 or 8 (got %d)", G);
  if (d->num_segments < 1 || d->num_segments > GQA_MAX_SEGMENTS)
    return capi_fail(MOE_EINVAL, "1..4 KV segments required");
  if (d->len[d->num_segments - 1] != d->T)
    return capi_fail(MOE_EINVAL, "the current segment must have T = %d tokens", d->T);
  for (int s = 0; s < d->num_segments; ++s) {
    if (d->len[s] < 0) return capi_fail(MOE_EINVAL, "segment %d has negative length", s);
    if (d->len[s] == 0) continue;
    if (!d->k[s] || !d->v[s] || !aligned16(d->k[s]) || !aligned16(d->v[s]))
      return capi_fail(MOE_EINVAL, "segment %d k/v must be non-null and 16-byte aligned", s);
    const int64_t minst = (int64_t)d->Hkv * 128;
    if (d->k_stride[s] < minst || d->v_stride[s] < minst || d->k_stride[s] % 8 ||
        d->v_stride[s] % 8)
      return capi_fail(MOE_EINVAL, "segment %d token stride must be >= %lld and a multiple of 8",
                       s, (long long)minst);
    // The kernels address up to 64 consecutive rows with 32-bit byte offsets.
    if (d->k_stride[s] > kMaxTokenStride || d->v_stride[s] > kMaxTokenStride)
      return capi_fail(MOE_EINVAL, "segment %d token stride must be <= %lld elements", s,
                       (long long)kMaxTokenStride);
  }
  if (d->T > 0 && (!d->q || !d->out || !aligned16(d->q) || !aligned16(d->out)))
    return capi_fail(MOE_EINVAL, "q/out must be non-null and 16-byte aligned");
  if ((long long)d->T * d->Hq * 128 >= (1LL << 31))
    return capi_fail(MOE_EINVAL, "T * Hq * 128 must be < 2^31");
  *shape = moe::gqa_shape(d->len, d->num_segments, d->Hq, d->Hkv, num_cus);
  return MOE_OK;
}

int device_cus(int *device, int *cus) {
  hipError_t e = hipGetDevice(device);
  if (e == hipSuccess) e = hipDeviceGetAttribute(cus, hipDeviceAttributeMultiprocessorCount, *device);
  if (e != hipSuccess) return moe::capi_fail(MOE_EDEVICE, "device query: %s", hipGetErrorString(e));
  return MOE_OK;
}

constexpr int kMaxGroup = 64;

int validate_heads(int Hq, int Hkv, int D, int dtype) {
  using moe::capi_fail;
  if (D != 64 && D != 128) return capi_fail(MOE_EINVAL, "head_dim must be 64 or 128 (got %d)", D);
  if (Hkv < 1 || Hq < 1 || Hq % Hkv || Hq / Hkv > kMaxGroup || Hq > (1 << 16))
    return capi_fail(MOE_EINVAL, "Hq must be a positive multiple of Hkv, at most %d times it (got %d, %d)", kMaxGroup, Hq,
                     Hkv);
  if (dtype != GQA_BF16 && dtype != GQA_FP16) return capi_fail(MOE_EINVAL, "unknown dtype %d", dtype);
  return MOE_OK;
}

int check_stride(const char *what, int64_t stride, int64_t least) {
  if (stride < least || stride > kMaxTokenStride || stride % 8)
    return moe::capi_fail(MOE_EINVAL, "%s must be in [%lld, %lld] and a multiple of 8 (got %lld)", what, (long long)least,
                          (long long)kMaxTokenStride, (long long)stride);
  return MOE_OK;
}

float scale_or_default(float scale, int D) {
  return scale > 0.f && scale < INFINITY ? scale : 1.0f / sqrtf((float)D);
}

int validate_packed_sizes(const gqa_packed_desc *d) {
  using moe::capi_fail;
  if (!d) return capi_fail(MOE_EINVAL, "null descriptor");
  if (const int rc = validate_heads(d->Hq, d->Hkv, d->D, d->dtype)) return rc;
  if (d->S < 0 || d->S > (1 << 20)) return capi_fail(MOE_EINVAL, "S must be in [0, 2^20] (got %d)", d->S);
  // The kernel divides numbers of query rows below 2^26; a grid has fewer than 2^32
  // threads, 256 per 128 query rows and per sequence, for every KV head.
  const int64_t rows = (int64_t)d->N * (d->Hq / d->Hkv);
  if (d->N < 0 || rows >= (1LL << 26) - 256 ||
      (rows / 128 + (d->S < d->N ? d->S : d->N) + 8) * d->Hkv >= (1LL << 24) - 8)
    return capi_fail(MOE_EINVAL,
                     "N must be >= 0, N * Hq / Hkv below 2^26 - 256 and N * Hq / 128 + S * Hkv below 2^24 (got N %d, S %d)",
                     d->N, d->S);
  return MOE_OK;
}

int validate_packed(const gqa_packed_desc *d) {
  using moe::capi_fail;
  if (const int rc = validate_packed_sizes(d)) return rc;
  if (d->N == 0 || d->S == 0) return MOE_OK;
  if (!d->q || !d->k || !d->v || !d->out || !aligned16(d->q) || !aligned16(d->k) || !aligned16(d->v) || !aligned16(d->out))
    return capi_fail(MOE_EINVAL, "q/k/v/out must be non-null and 16-byte aligned");
  if (!d->starts || ((uintptr_t)d->starts & 3u)) return capi_fail(MOE_EINVAL, "starts must be given");
  int rc = check_stride("q token stride", d->q_stride, (int64_t)d->Hq * d->D);
  if (!rc) rc = check_stride("k token stride", d->k_stride, (int64_t)d->Hkv * d->D);
  if (!rc) rc = check_stride("v token stride", d->v_stride, (int64_t)d->Hkv * d->D);
  return rc;
}

size_t packed_workspace(const gqa_packed_desc *d) { return moe::gqa_packed_workspace(d->N, d->Hq, d->Hkv, d->S); }

int validate_paged_sizes(const gqa_paged_desc *d) {
  using moe::capi_fail;
  if (!d) return capi_fail(MOE_EINVAL, "null descriptor");
  if (const int rc = validate_heads(d->Hq, d->Hkv, d->D, d->dtype)) return rc;
  if (d->B < 0 || d->B > (1 << 16)) return capi_fail(MOE_EINVAL, "B must be in [0, 2^16] (got %d)", d->B);
  if (d->page < 16 || d->page > 1024 || d->page % 16)
    return capi_fail(MOE_EINVAL, "page must be a multiple of 16 up to 1024 (got %d)", d->page);
  if (d->P < 1 || d->M < 1 || (int64_t)d->M * d->page >= 1LL << 31)
    return capi_fail(MOE_EINVAL, "P and M must be positive and M * page < 2^31 (got %d, %d)", d->P, d->M);
  // 32-key steps over all sequences and blocks of 16 query heads are counted in 32 bits.
  const int64_t steps = (int64_t)d->B * d->Hkv * ((d->Hq / d->Hkv + 15) / 16);
  if (steps >= 1LL << 24)  // (a grid has fewer than 2^32 threads)
    return capi_fail(MOE_EINVAL, "B * Hkv * ceil(Hq / Hkv / 16) must be below 2^24 (got B %d, Hkv %d)", d->B, d->Hkv);
  if (steps > (1LL << 30) / (((int64_t)d->M * d->page + 31) / 32))
    return capi_fail(MOE_EINVAL, "B * Hkv * M * page / 32 must be at most 2^30 (B %d, Hkv %d, M %d, page %d)", d->B,
                     d->Hkv, d->M, d->page);
  return MOE_OK;
}

int validate_paged(const gqa_paged_desc *d) {
  using moe::capi_fail;
  if (const int rc = validate_paged_sizes(d)) return rc;
  if (d->B == 0) return MOE_OK;
  if (!d->q || !d->k || !d->v || !d->out || !aligned16(d->q) || !aligned16(d->k) || !aligned16(d->v) || !aligned16(d->out))
    return capi_fail(MOE_EINVAL, "q/k/v/out must be non-null and 16-byte aligned");
  if (!d->tables || !d->lengths || ((uintptr_t)d->tables & 3u) || ((uintptr_t)d->lengths & 3u))
    return capi_fail(MOE_EINVAL, "tables and lengths must be given");
  if (d->table_stride < d->M) return capi_fail(MOE_EINVAL, "table_stride must be at least M = %d", d->M);
  int rc = check_stride("q row stride", d->q_stride, (int64_t)d->Hq * d->D);
  for (int kv = 0; !rc && kv < 2; ++kv) {
    const int64_t *st = kv ? d->v_strides : d->k_strides;
    if (st[0] < 8 || st[0] % 8 || st[1] < 8 || st[1] % 8)
      return capi_fail(MOE_EINVAL, "page and head strides must be positive multiples of 8");
    rc = check_stride("page row stride", st[2], d->D);
  }
  return rc;
}

size_t paged_workspace(const gqa_paged_desc *d, int cus) {
  return moe::gqa_paged_workspace(d->B, d->Hq, d->Hkv, d->D, (int64_t)d->M * d->page, cus);
}

int need_workspace(const void *workspace, size_t have, size_t need) {
  if (!workspace || !aligned16(workspace) || have < need)
    return moe::capi_fail(MOE_ESPACE, "workspace has %zu bytes, needs %zu, 16-byte aligned", have, need);
  return MOE_OK;
}

// Runs `launch` with a plan's device current.
template <typename F>
int on_device(int device, const char *what, F launch) {
  int prev = -1;
  hipError_t e = hipGetDevice(&prev);
  if (e == hipSuccess && prev != device) e = hipSetDevice(device);
  if (e == hipSuccess) e = launch();
  if (prev >= 0 && prev != device) (void)hipSetDevice(prev);
  if (e != hipSuccess) return moe::capi_fail(MOE_EDEVICE, "%s: %s", what, hipGetErrorString(e));
  return MOE_OK;
}

}  // namespace

extern "C" {

int gqa_packed_workspace_bytes(const gqa_packed_desc *d, size_t *bytes) {
  if (const int rc = validate_packed_sizes(d)) return rc;
  if (!bytes) return moe::capi_fail(MOE_EINVAL, "null bytes");
  *bytes = packed_workspace(d);
  return MOE_OK;
}

int gqa_packed_plan_create(gqa_packed_plan **out, const gqa_packed_desc *d) {
  if (!out) return moe::capi_fail(MOE_EINVAL, "null plan pointer");
  *out = nullptr;
  int rc = validate_packed(d), dev = 0, cus = 0;
  if (!rc) rc = need_workspace(d->workspace, d->workspace_bytes, packed_workspace(d));
  if (!rc) rc = device_cus(&dev, &cus);
  if (rc) return rc;
  gqa_packed_plan *p = new (std::nothrow) gqa_packed_plan;
  if (!p) return moe::capi_fail(MOE_EINVAL, "out of host memory");
  p->a = moe::GqaPackedArgs{(const uint16_t *)d->q, (const uint16_t *)d->k, (const uint16_t *)d->v, (uint16_t *)d->out,
                            d->starts, d->q_stride, d->k_stride, d->v_stride, d->N, d->S, d->Hq, d->Hkv, d->D, d->dtype,
                            scale_or_default(d->scale, d->D), nullptr, nullptr, nullptr, nullptr, 0, 0, 0, 0, 0, 0, 0};
  moe::gqa_packed_bind(&p->a, d->workspace);
  moe::gqa_packed_constants(&p->a);
  p->device = dev;
  p->cus = cus;
  *out = p;
  return MOE_OK;
}

int gqa_packed_plan_run(gqa_packed_plan *p, void *stream) {
  if (!p) return moe::capi_fail(MOE_EINVAL, "null plan");
  if (p->a.N == 0 || p->a.S == 0) return MOE_OK;
  return on_device(p->device, "packed gqa launch", [&] { return moe::launch_gqa_packed(p->a, p->cus, (hipStream_t)stream); });
}

int gqa_packed_plan_read_status(gqa_packed_plan *p, void *stream, uint32_t *flags) {
  if (!p || !flags) return moe::capi_fail(MOE_EINVAL, "null plan or flags");
  return on_device(p->device, "status",
                   [&] { return moe::read_and_clear_status(p->a.status, flags, (hipStream_t)stream); });
}

void gqa_packed_plan_destroy(gqa_packed_plan *p) { delete p; }

int gqa_paged_workspace_bytes(const gqa_paged_desc *d, size_t *bytes) {
  int rc = validate_paged_sizes(d), dev = 0, cus = 0;
  if (!rc && !bytes) rc = moe::capi_fail(MOE_EINVAL, "null bytes");
  if (!rc) rc = device_cus(&dev, &cus);
  if (!rc) *bytes = paged_workspace(d, cus);
  return rc;
}

int gqa_paged_plan_create(gqa_paged_plan **out, const gqa_paged_desc *d) {
  if (!out) return moe::capi_fail(MOE_EINVAL, "null plan pointer");
  *out = nullptr;
  int rc = validate_paged(d), dev = 0, cus = 0;
  if (!rc) rc = need_workspace(d->workspace, d->workspace_bytes, 256);
  if (!rc) rc = device_cus(&dev, &cus);
  if (!rc) rc = need_workspace(d->workspace, d->workspace_bytes, paged_workspace(d, cus));
  if (rc) return rc;
  gqa_paged_plan *p = new (std::nothrow) gqa_paged_plan;
  if (!p) return moe::capi_fail(MOE_EINVAL, "out of host memory");
  p->a = moe::GqaPagedArgs{(const uint16_t *)d->q, (const uint16_t *)d->k, (const uint16_t *)d->v, (uint16_t *)d->out,
                           d->tables, d->lengths, d->q_stride, d->table_stride, d->k_strides[0], d->k_strides[1],
                           d->k_strides[2], d->v_strides[0], d->v_strides[1], d->v_strides[2], d->B, d->Hq, d->Hkv, d->D,
                           d->P, d->page, d->M, d->dtype, scale_or_default(d->scale, d->D), nullptr, nullptr, nullptr};
  moe::gqa_paged_bind(&p->a, d->workspace);
  p->device = dev;
  p->cus = cus;
  *out = p;
  return MOE_OK;
}

int gqa_paged_plan_run(gqa_paged_plan *p, void *stream) {
  if (!p) return moe::capi_fail(MOE_EINVAL, "null plan");
  if (p->a.B == 0) return MOE_OK;
  return on_device(p->device, "paged gqa launch", [&] { return moe::launch_gqa_paged(p->a, p->cus, (hipStream_t)stream); });
}

int gqa_paged_plan_read_status(gqa_paged_plan *p, void *stream, uint32_t *flags) {
  if (!p || !flags) return moe::capi_fail(MOE_EINVAL, "null plan or flags");
  return on_device(p->device, "status",
                   [&] { return moe::read_and_clear_status(p->a.status, flags, (hipStream_t)stream); });
}

void gqa_paged_plan_destroy(gqa_paged_plan *p) { delete p; }

int gqa_seg_workspace_bytes(const gqa_seg_desc *d, size_t *bytes) {
  int dev = 0, cus = 0;
  moe::GqaShape shape{1, 4, 2, false};
  int rc = device_cus(&dev, &cus);
  if (rc) return rc;
  if ((rc = validate(d, cus, &shape))) return rc;
  if (!bytes) return moe::capi_fail(MOE_EINVAL, "null bytes");
  // At least what the short-chunk kernel needs, which does not depend on the
  // history: a workspace sized with any history then serves every other.
  const size_t own = moe::gqa_partial_bytes(d->T, d->Hq, shape.nsplit);
  const size_t any = moe::gqa_partial_bytes(d->T, d->Hq, moe::gqa_short_shape(d->T, d->Hq, d->Hkv, cus).nsplit);
  *bytes = own > any ? own : any;
  return MOE_OK;
}

int gqa_seg_choice(const gqa_seg_desc *d, int32_t num_cus, int32_t out[2]) {
  moe::GqaShape shape{1, 4, 2, false};
  if (const int rc = validate(d, num_cus, &shape)) return rc;
  if (!out || num_cus < 1) return moe::capi_fail(MOE_EINVAL, "null output or no compute units");
  out[0] = shape.prefill;
  out[1] = shape.nsplit;
  return MOE_OK;
}

int gqa_seg_plan_create(gqa_seg_plan **out, const gqa_seg_desc *d) {
  if (!out) return moe::capi_fail(MOE_EINVAL, "null plan pointer");
  *out = nullptr;
  int dev = 0, cus = 0;
  moe::GqaShape shape{1, 4, 2, false};
  int rc = device_cus(&dev, &cus);
  if (rc) return rc;
  if ((rc = validate(d, cus, &shape))) return rc;
  size_t need = moe::gqa_partial_bytes(d->T, d->Hq, shape.nsplit);
  auto lacks = [&] { return need && (d->workspace_bytes < need || !d->workspace || !aligned16(d->workspace)); };
  if (shape.prefill && lacks()) {
    // Less workspace than gqa_seg_workspace_bytes() asks for: the short-chunk
    // kernel needs none at these lengths, or less.
    shape = moe::gqa_short_shape(d->T, d->Hq, d->Hkv, cus);
    need = moe::gqa_partial_bytes(d->T, d->Hq, shape.nsplit);
  }
  if (lacks())
    return moe::capi_fail(MOE_ESPACE, "workspace has %zu bytes, needs %zu", d->workspace_bytes,
                          need);
  gqa_seg_plan *p = new (std::nothrow) gqa_seg_plan;
  if (!p) return moe::capi_fail(MOE_EINVAL, "out of host memory");
  moe::GqaArgs &a = p->a;
  a.q = (const uint16_t *)d->q;
  a.out = (uint16_t *)d->out;
  a.num_segments = d->num_segments;
  a.history = 0;
  for (int s = 0; s < moe::kGqaMaxSegments; ++s) {
    const bool live = s < d->num_segments;
    a.k[s] = live ? (const uint16_t *)d->k[s] : nullptr;
    a.v[s] = live ? (const uint16_t *)d->v[s] : nullptr;
    a.k_stride[s] = live ? d->k_stride[s] : 0;
    a.v_stride[s] = live ? d->v_stride[s] : 0;
    a.len[s] = live ? d->len[s] : 0;
    if (live && s < d->num_segments - 1) a.history += d->len[s];
  }
  a.T = d->T;
  a.Hq = d->Hq;
  a.Hkv = d->Hkv;
  a.scale = (d->scale > 0.f && d->scale < INFINITY) ? d->scale : 1.0f / sqrtf((float)d->D);
  a.partial = (float *)d->workspace;
  p->shape = shape;
  p->device = dev;
  *out = p;
  return MOE_OK;
}

int gqa_seg_plan_run(gqa_seg_plan *p, void *stream) {
  if (!p) return moe::capi_fail(MOE_EINVAL, "null plan");
  if (p->a.T == 0) return MOE_OK;
  int prev = -1;
  hipError_t e = hipGetDevice(&prev);
  if (e == hipSuccess && prev != p->device) e = hipSetDevice(p->device);
  if (e == hipSuccess) e = moe::launch_gqa(p->a, p->shape, (hipStream_t)stream);
  if (prev >= 0 && prev != p->device) (void)hipSetDevice(prev);
  if (e != hipSuccess) return moe::capi_fail(MOE_EDEVICE, "gqa launch: %s", hipGetErrorString(e));
  return MOE_OK;
}

void gqa_seg_plan_destroy(gqa_seg_plan *p) { delete p; }

}  // extern "C"
