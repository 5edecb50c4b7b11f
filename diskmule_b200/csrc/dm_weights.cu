// dm_weights.cu -- the attention that each cached token has received (include/diskmule_attention.h).
//
// w[k] += sum over query rows r of 2^(scale q_r k - lse_r), scale and lse times log2 e: the weights
// of attention again, from its statistics, summed along the other axis. So keys are the rows of
// the products here (mma.sync tiles of 16 keys x 8 query rows): a key's sum stays in the threads
// that hold its row, over all queries and heads, and one block owns a key, so nothing is added
// atomically and the order of the sums is fixed.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "dm_attention.cuh"
#include "dm_attention_tc.cuh"
#include "dm_mma.cuh"
#include "dm_tcgen05.cuh"

using dmi::fail;
namespace cg = cooperative_groups;

namespace dma {

using namespace dm::tc;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kWarpKeys = 16;               // pages are multiples of it
constexpr int kKeys = kWarps * kWarpKeys;   // of a block
constexpr int kTileRows = 8;                // query rows of a product
constexpr int kMostRanks = 8;               // blocks of a cluster, which share the keys' queries

template <int DP>
struct Cfg {
  static constexpr int kStages = DP == 256 ? 2 : 4;           // heads of a warp's keys
  static constexpr int kTiles = DP == 256 ? 4 : 8;            // query tiles of a step
  static constexpr int kChunk = kWarpKeys * DP * 2;           // bytes
  static constexpr int kTile = kTileRows * DP * 2;
  static constexpr int kRing = kStages * kChunk;
  static constexpr int kStep = kTiles * kTile;
  static constexpr int kSmem = 1024 + kWarps * kRing + 2 * kStep;
};

struct WeightsArgs {
  const uint16_t *q;
  const float *lse;
  int64_t q_stride[2];
  const int32_t *offsets;
  float *weights;
  int64_t weights_stride, tokens;
  int32_t heads, group, window, sinks;
  float scale;  // times log2 e
  DecodeArgs d;  // rows, max_length, waits
};

template <int DP, bool BF16>
__global__ void __launch_bounds__(kThreads)
weights_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ WeightsArgs a,
               const __grid_constant__ KvView c) {
  using C = Cfg<DP>;
  constexpr unsigned kAll = 0xffffffffu;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[kWarps][C::kStages];
  __shared__ float lse_of[2][C::kTiles * kTileRows];
  __shared__ float sums[kMostRanks][kKeys];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
  const uint32_t ring = base + warp * C::kRing, q_at = base + kWarps * C::kRing;
  auto cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
  if (tid < kWarps * C::kStages) mbar_init(smem_u32(&full[tid / C::kStages][tid % C::kStages]), 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  wait_for_previous();
  let_next_start();

  // ---- the entry, its queries and this block's keys
  const int entry = blockIdx.y, dim = c.head_dim, group = a.group;
  const int64_t q0 = min((int64_t)max(a.offsets[entry], 0), a.tokens);
  const int lq = (int)(max(q0, min((int64_t)a.offsets[entry + 1], a.tokens)) - q0);
  int length;
  const int row = sequence_of(c, a.d, entry, &length);
  const int first = blockIdx.x / ranks * kKeys, key = first + warp * kWarpKeys;
  const int end = (int)min((int64_t)length, a.weights_stride);
  const int p0 = length - lq;  // place of the first query
  // seen by the first query's window, or by all
  const bool seen = !a.window || first + kKeys > max(p0, 0) - (a.window - 1) || first < a.sinks;
  int twice = 0;
  if (a.d.sequences && lq > 0)
    for (int i = tid; i < entry; i += kThreads) twice |= a.d.sequences[i] == row;
  twice = __syncthreads_or(twice);
  if (twice && first == 0 && rank == 0 && tid == 0 && length > 0) atomicOr(c.status, DM_KV_BAD_SEQUENCE);
  if (lq == 0 || first >= end || !seen || twice) return;  // all ranks alike
  if (ranks > 1) cluster.sync();  // the others' shared memory is there

  // ---- tiles of query rows, of all key/value heads one after the other; this block's share
  const int rows = lq * group;  // at most 2^31 by the call's check
  const int per_head = (rows + kTileRows - 1) / kTileRows;
  const int64_t all = (int64_t)per_head * c.kv_heads;
  const int u0 = (int)(all * rank / ranks), u1 = (int)(all * (rank + 1) / ranks);
  const int h0 = u0 / per_head, h1 = (u1 + per_head - 1) / per_head;
  const bool working = key < end && u1 > u0;  // of this warp

  // ---- keys: a head of the warp's 16 at a time
  const int page = key < end ? c.table[(int64_t)row * c.max_pages + key / c.page_tokens] : 0;
  if (key < end && (unsigned)page >= (unsigned)c.pages && lane == 0) atomicOr(c.status, DM_KV_BAD_TOKEN);
  auto at = [](int slab, int r, int v) { return (uint32_t)((v >> 3) * slab + r * 128 + ((v ^ r) & 7) * 16); };
  int loads = h0;
  auto load_keys = [&]() {
    if (working && loads < h1) {
      const int stage = (loads - h0) % C::kStages;
      const uint32_t bar = smem_u32(&full[warp][stage]);
      if (lane == 0) mbar_expect_tx(bar, C::kChunk);
      __syncwarp();
      if (lane < DP / 64)
        tma_load_4d(ring + stage * C::kChunk + lane * kWarpKeys * 128, &k_map, lane * 64, key & (c.page_tokens - 1),
                    loads, page, bar);
    }
    loads++;
  };
  for (int s = 0; s < C::kStages; s++) load_keys();

  // ---- queries and their statistics: kTiles tiles a step, two steps in turn
  constexpr int kVec = DP / 8;
  auto load_queries = [&](int u, int buffer) {
    for (int i = tid; i < C::kTiles * kTileRows * kVec; i += kThreads) {
      const int r = i / kVec, v = i % kVec;
      const int tile = u + r / kTileRows, head = tile / per_head;
      const int at_row = (tile - head * per_head) * kTileRows + r % kTileRows;
      const bool valid = tile < u1 && at_row < rows && v < dim / 8;
      const int64_t token = q0 + at_row / group;
      const int of = head * group + at_row % group;
      cp16(q_at + buffer * C::kStep + r / kTileRows * C::kTile + at(1024, r % kTileRows, v),
           valid ? a.q + token * a.q_stride[0] + of * a.q_stride[1] + v * 8 : a.q, valid);
      if (v == 0) lse_of[buffer][r] = valid ? a.lse[token * a.heads + of] : -INFINITY;
    }
    asm volatile("cp.async.commit_group;");
  };
  load_queries(u0, 0);

  float total[2] = {0.0f, 0.0f};
  uint32_t kf[DP / 16][4];
  int held = -1;  // the head whose keys are in registers
  bool alive = true;
  int buffer = 0;
  for (int u = u0; u < u1; u += C::kTiles, buffer ^= 1) {
    asm volatile("cp.async.wait_group 0;");
    __syncthreads();  // this step is there, and all have left the other
    if (u + C::kTiles < u1) load_queries(u + C::kTiles, buffer ^ 1);
    if (!working) continue;
    float part[2] = {0.0f, 0.0f};
    for (int t = 0; t < C::kTiles && u + t < u1; t++) {
      const int head = (u + t) / per_head, tile = u + t - head * per_head;
      if (head != held) {
        held = head;
        const int stage = (head - h0) % C::kStages;
        const uint32_t parity = ((head - h0) / C::kStages) & 1;
        if (alive && !__all_sync(kAll, copy_landed(smem_u32(&full[warp][stage]), parity, a.d.wait_limit))) {
          if (lane == 0) atomicExch(a.d.timeout, 1);
          // the copies in flight land before the block ends
          for (int h = head; h < min(loads, h1); h++)
            mbar_wait(smem_u32(&full[warp][(h - h0) % C::kStages]), ((h - h0) / C::kStages) & 1);
          alive = false;
        }
        const int r = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
        for (int k = 0; k < DP / 16; k++) ldm4(ring + stage * C::kChunk + at(kWarpKeys * 128, r, 2 * k + (lane >> 4)), kf[k]);
        __syncwarp();
        if (alive) load_keys();
      }
      // places of the tile's first and last row
      const int from = p0 + tile * kTileRows / group, to = p0 + min(rows - 1, tile * kTileRows + kTileRows - 1) / group;
      const bool window_hides = a.window && key + kWarpKeys <= max(from, 0) - (a.window - 1) && key >= a.sinks;
      if (key > to || window_hides) continue;
      float s[4] = {}, s2[4] = {};
      const uint32_t qt = q_at + buffer * C::kStep + t * C::kTile;
#pragma unroll
      for (int k = 0; k < DP / 32; k++) {
        uint32_t b[4];
        ldm4(qt + at(1024, lane & 7, 4 * k + (lane >> 3)), b);
        mma16816<BF16>(s, kf[2 * k], b[0], b[1]);
        mma16816<BF16>(s2, kf[2 * k + 1], b[2], b[3]);
      }
      const float2 lse = *reinterpret_cast<const float2 *>(&lse_of[buffer][t * kTileRows + (lane & 3) * 2]);
      const float z[2] = {lse.x == -INFINITY ? -INFINITY : -lse.x * kLog2e,
                          lse.y == -INFINITY ? -INFINITY : -lse.y * kLog2e};
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; i++) w[i] = exp2_fast(fmaf(s[i] + s2[i], a.scale, z[i & 1]));
      // some key is hidden from some row
      if (key + kWarpKeys - 1 > from || (a.window && to - key >= a.window && key + kWarpKeys > a.sinks)) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int r = tile * kTileRows + (lane & 3) * 2 + (i & 1);
          const int p = p0 + r / group, j = key + (lane >> 2) + (i >> 1) * 8;
          const bool sees = r < rows && j <= p && (!a.window || (unsigned)p - j < (unsigned)a.window || j < a.sinks);
          w[i] = sees ? w[i] : 0.0f;
        }
      }
      part[0] += w[0] + w[1];
      part[1] += w[2] + w[3];
    }
    total[0] += part[0];
    total[1] += part[1];
  }
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) total[i] += __shfl_xor_sync(kAll, total[i], x);
  if (ranks > 1) {
    float *there = cluster.map_shared_rank(&sums[0][0], 0) + rank * kKeys + warp * kWarpKeys;
    if ((lane & 3) == 0) there[lane >> 2] = total[0], there[(lane >> 2) + 8] = total[1];
    cluster.sync();
    if (rank == 0 && tid < kKeys && first + tid < end) {
      float sum = 0.0f;
      for (int i = 0; i < ranks; i++) sum += sums[i][tid];
      a.weights[row * a.weights_stride + first + tid] += sum;
    }
  } else if ((lane & 3) == 0) {
    for (int i = 0; i < 2; i++) {
      const int j = key + (lane >> 2) + i * 8;
      if (j < end) a.weights[row * a.weights_stride + j] += total[i];
    }
  }
}

template <int DP, bool BF16>
int32_t launch_weights(dim3 grid, int ranks, const CUtensorMap &map, const WeightsArgs &a, const KvView &c,
                       cudaStream_t s) {
  auto fn = weights_kernel<DP, BF16>;
  DM_CUDA(dm::ensure_smem_limit((const void *)fn), "attention shared memory");
  return launch_clusters("weights launch", fn, grid, ranks, kThreads, Cfg<DP>::kSmem, s, map, a, c);
}

}  // namespace
}  // namespace dma

using namespace dma;

extern "C" int32_t dm_attention_weights(dm_kv_cache *cache, const dm_attention_weights_desc *in, void *stream) {
  if (!cache || !in) return fail(DM_ERR_INVALID_ARGUMENT, "null argument");
  const dm_kv_cache_desc &d = cache->desc;
  if (in->heads <= 0 || in->heads % d.kv_heads || in->heads / d.kv_heads > 128)
    return fail(DM_ERR_ELEMENT_COUNT, "%d query heads over %d key/value heads", in->heads, d.kv_heads);
  if (in->layer < 0 || in->layer >= d.layers) return fail(DM_ERR_INVALID_LAYER, "layer %d of %d", in->layer, d.layers);
  if (in->sequences < 0 || in->sequences > 65535) return fail(DM_ERR_ELEMENT_COUNT, "%d sequences", in->sequences);
  if (in->window < 0 || in->sinks < 0)
    return fail(DM_ERR_ELEMENT_COUNT, "window %d, %d sinks", in->window, in->sinks);
  if (in->max_length < 0) return fail(DM_ERR_ELEMENT_COUNT, "max_length %d", in->max_length);
  if (in->tokens < 0 || in->tokens > kMostTokens) return fail(DM_ERR_ELEMENT_COUNT, "a bad number of tokens");
  if (in->tokens * in->heads > INT32_MAX) return fail(DM_ERR_OVERFLOW, "too many query rows");
  if (in->weights_stride < 0) return fail(DM_ERR_INVALID_ARGUMENT, "a negative stride of weights");
  const int64_t keys = std::min(std::min<int64_t>(in->max_length, (int64_t)d.max_pages * d.page_tokens), in->weights_stride);
  if (in->tokens == 0 || in->sequences == 0 || keys == 0) return DM_OK;
  if (!in->q || !in->lse || !in->offsets || !in->weights) return fail(DM_ERR_INVALID_ARGUMENT, "null tensor");
  if ((uintptr_t)in->q & 15) return fail(DM_ERR_INVALID_ARGUMENT, "attention tensors must be 16-byte aligned");
  if (((uintptr_t)in->lse | (uintptr_t)in->weights) & 3)
    return fail(DM_ERR_INVALID_ARGUMENT, "lse and weights must be 4-byte aligned");
  WeightsArgs a{};
  if (int32_t rc = check_strides(in->q_stride, in->heads, d.head_dim, a.q_stride, "query")) return rc;
  if (int32_t rc = check_scale(in->scale, d.head_dim, &a.scale)) return rc;
  a.q = (const uint16_t *)in->q;
  a.lse = in->lse;
  a.offsets = in->offsets;
  a.weights = in->weights;
  a.weights_stride = in->weights_stride;
  a.tokens = in->tokens;
  a.heads = in->heads;
  a.group = in->heads / d.kv_heads;
  a.window = in->window;
  a.sinks = in->sinks;
  a.d.sequences = in->rows;
  a.d.max_length = (int32_t)std::min<int64_t>(in->max_length, (int64_t)d.max_pages * d.page_tokens);
  a.d.timeout = cache->ctx->status + kStatusWord;
  a.d.wait_limit = wait_limit(cache->ctx);
  cudaSetDevice(cache->ctx->device);
  CUtensorMap maps[2];
  if (!describe_chunks(d.type, cache->view, in->layer, kWarpKeys, maps))
    return fail(DM_ERR_COMMAND, "could not describe the cache for TMA");
  const int64_t tiles = (keys + kKeys - 1) / kKeys;
  // few blocks: several share the queries of their keys
  int ranks = 1;
  const int64_t steps = std::max<int64_t>(1, in->tokens * a.group / (kTileRows * in->sequences)) * d.kv_heads;
  while (ranks < kMostRanks && tiles * in->sequences * ranks < 2 * 148 && steps >= 2 * ranks) ranks *= 2;
  const dim3 grid((unsigned)(tiles * ranks), in->sequences);
  cudaStream_t s = (cudaStream_t)stream;
  const bool bf = d.type == DM_BF16;
  if (d.head_dim <= 64)
    return bf ? launch_weights<64, true>(grid, ranks, maps[0], a, cache->view, s)
              : launch_weights<64, false>(grid, ranks, maps[0], a, cache->view, s);
  if (d.head_dim <= 128)
    return bf ? launch_weights<128, true>(grid, ranks, maps[0], a, cache->view, s)
              : launch_weights<128, false>(grid, ranks, maps[0], a, cache->view, s);
  return bf ? launch_weights<256, true>(grid, ranks, maps[0], a, cache->view, s)
            : launch_weights<256, false>(grid, ranks, maps[0], a, cache->view, s);
}
