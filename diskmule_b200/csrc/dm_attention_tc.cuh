// dm_attention_tc.cuh -- attention on tcgen05 tiles (dm_attention_tc.cu).
#pragma once

#include <cuda.h>

#include "dm_attention.cuh"

namespace dma {

// Whole prompts. The tensors need strides that a tensor map can hold.
bool tile_prompt_fits(const PromptArgs &p);
int32_t launch_tile_prompt(int32_t type, const PromptArgs &p, dm_cuda_context *ctx, cudaStream_t stream);
int64_t wait_limit(const dm_cuda_context *ctx);  // of a bounded wait, clocks

// The shared part of a decode call, in d.splits parts, or twice as many where the two units
// of a block alternate.
int tile_keys(int dim);  // keys of a tile
bool tile_shared_alternates(int dim, int group, int batch);
int tile_shared_items(int dim, int kv_heads, int group, int batch);
int32_t launch_tile_shared(int32_t type, const DecodeArgs &d, const KvView &c, cudaStream_t stream);

// Tensor maps of a cache layer's K and V with boxes of 64 values and `rows` tokens of a page.
bool describe_chunks(int32_t type, const KvView &c, int layer, int rows, CUtensorMap *maps);

}  // namespace dma
