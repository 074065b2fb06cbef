// Internal launch interface of the norm and rotation of queries and keys.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_internal.h"

namespace moe {

struct QkArgs {
  int N, Hq, Hkv, D, R, f16, interleaved, weights_fp32;
  const uint16_t *q, *k, *v;
  const int32_t *positions;
  const float *inv_freq;
  const void *q_weight, *k_weight;
  uint16_t *q_out, *k_out;
  int64_t q_stride, k_stride, v_stride;
  float eps;
  int layer;
  bool cached;  // keys and values go to the slots of `cache` too
  KvState cache;
};
hipError_t launch_qk_norm_rope(const QkArgs &a, int cus, hipStream_t s);

}  // namespace moe
