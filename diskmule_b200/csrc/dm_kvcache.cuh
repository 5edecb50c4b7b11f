// dm_kvcache.cuh -- the paged key/value cache's host object and device view
// (include/diskmule_attention.h).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/diskmule_attention.h"
#include "dm_internal.cuh"

namespace dma {

// Tokens of a sequence or a packed tensor at most: kernels step past the last one by up to a few
// hundred, in 32 bits.
constexpr int32_t kMostTokens = INT32_MAX - 4096;

// What kernels see of a cache. Byte strides; every row of head_dim values is 16-byte aligned.
struct KvView {
  uint8_t *memory;
  int32_t *table, *lengths, *references;
  int32_t *status;
  int32_t layers, kv_heads, head_dim, page_tokens, pages, max_sequences, max_pages;
  int64_t page_bytes, layer_bytes, head_bytes;  // of a page, of its layer (K and V), of one head
};

// The next kernel on the stream may be scheduled (it then waits, below).
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
// Wait until the kernel before this one on the stream has ended and its writes are seen.
__device__ __forceinline__ void wait_for_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// A launch that may be scheduled while the kernel before it still runs; the kernel calls
// wait_for_previous before it touches what that one or its predecessors wrote.
template <typename... Params, typename... Args>
int32_t launch_chained(const char *what, void (*kernel)(Params...), dim3 grid, int threads, size_t smem,
                       cudaStream_t stream, const Args &...args) {
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = threads;
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = 1;
  DM_CUDA(cudaLaunchKernelEx(&config, kernel, args...), what);
  return DM_OK;
}

}  // namespace dma

struct dm_kv_cache {
  dm_cuda_context *ctx = nullptr;
  dm_kv_cache_desc desc{};
  dma::KvView view{};
  bool own_memory = false, own_table = false, own_lengths = false, own_references = false;
  // bookkeeping scratch: the plan of the call in flight (dm_kvcache.cu)
  int32_t *scratch = nullptr;
};
