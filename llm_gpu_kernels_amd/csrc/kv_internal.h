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
  // How k and v hold their rows (KV_STORAGE_*, 0: as 16-bit elements), and with it the
  // scales [layers, pages, kv_heads, head_dim / 32, page_size] and the tokens' type.
  int storage, f16;
  uint8_t *k_scales, *v_scales;
  // Bytes of a page of k or v in one layer, and of its scales (0: none).
  int64_t page_bytes, scale_page_bytes;
};

size_t kv_workspace_bytes(int pages);
void kv_bind_workspace(KvState *s, void *workspace);

hipError_t launch_kv_reserve(const KvState &s, const int32_t *counts, int stride, hipStream_t st);
hipError_t launch_kv_append(const KvState &s, int layer, const uint16_t *k, const uint16_t *v, int64_t k_stride,
                            int64_t v_stride, int n, hipStream_t st);
hipError_t launch_kv_gather(const KvState &s, int layer, const int32_t *rows, const int32_t *starts, int n, uint16_t *k,
                            uint16_t *v, int64_t k_stride, int64_t v_stride, int tokens, hipStream_t st);
hipError_t launch_kv_fork(const KvState &s, const int32_t *src, const int32_t *dst, int n, hipStream_t st);
hipError_t launch_kv_free(const KvState &s, const int32_t *rows, int n, hipStream_t st);
hipError_t launch_kv_compact(const KvState &s, hipStream_t st);

}  // namespace moe
