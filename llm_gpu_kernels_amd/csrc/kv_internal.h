// Internal launch interface of the paged key-value cache kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace moe {

struct KvState {
  int pages, page_size, kv_heads, head_dim, layers;
  int sequences, max_pages, max_tokens;
  uint16_t *k, *v;
  int32_t *tables, *lengths, *refs, *starts;
  int64_t *slots;
  uint32_t *status;
  // Scratch: the count of moves, the workgroups of a fork that have finished (0
  // between calls), the moves' source and target pages, the pages of a reserve in
  // order, and the number of a moved page's move.
  int32_t *num_moves, *arrived, *move_src, *move_dst, *list, *move_of;
};

size_t kv_workspace_bytes(int pages);
void kv_bind_workspace(KvState *s, void *workspace);

hipError_t launch_kv_reserve(const KvState &s, const int32_t *counts, int stride, hipStream_t st);
hipError_t launch_kv_append(const KvState &s, int layer, const uint16_t *k, const uint16_t *v, int64_t k_stride,
                            int64_t v_stride, int n, hipStream_t st);
hipError_t launch_kv_fork(const KvState &s, const int32_t *src, const int32_t *dst, int n, hipStream_t st);
hipError_t launch_kv_free(const KvState &s, const int32_t *rows, int n, hipStream_t st);
hipError_t launch_kv_compact(const KvState &s, hipStream_t st);

}  // namespace moe
