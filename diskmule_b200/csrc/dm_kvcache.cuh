// dm_kvcache.cuh -- the paged key/value cache's host object and device view
// (include/diskmule_attention.h).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/diskmule_attention.h"
#include "dm_internal.cuh"

namespace dma {

// What kernels see of a cache. Byte strides; every row of head_dim values is 16-byte aligned.
struct KvView {
  uint8_t *memory;
  int32_t *table, *lengths, *references;
  int32_t *status;
  int32_t layers, kv_heads, head_dim, page_tokens, pages, max_sequences, max_pages;
  int64_t page_bytes, layer_bytes, head_bytes;  // of a page, of its layer (K and V), of one head
};

}  // namespace dma

struct dm_kv_cache {
  dm_cuda_context *ctx = nullptr;
  dm_kv_cache_desc desc{};
  dma::KvView view{};
  bool own_memory = false, own_table = false, own_lengths = false, own_references = false;
  // bookkeeping scratch: the plan of the call in flight (dm_kvcache.cu)
  int32_t *scratch = nullptr;
};
