// dm_weights.cu -- the attention that each cached token has received (include/diskmule_attention.h).
//
// w[k] += sum over query rows r of 2^(scale q_r k - lse_r), scale and lse times log2 e: the weights
// of attention again, from its statistics, summed along the other axis. So keys are the rows of
// the products here (mma.sync tiles of 16 keys x 8 query rows): a key's sum stays in the threads
// that hold its row, over all queries and heads, and one block owns a key, so nothing is added
// atomically and the order of the sums is fixed.
//
// scale q k and lse may be in the tens where their difference is near 0, so neither may be rounded
// before it is taken. With c the f32 next to scale log2 e, the weight is 2^(c (q k - lse / scale)) to
// one part in 2^24 of the exponent; c lse / scale is kept as hi + lo, the exponent is one fused
// c q k - hi, and the factor 2^-lo goes into the sum's multiplication. (c lse / scale rounded to f32
// would be off by up to 2^-24 of itself, one part in a million of a weight where it is 24.)
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
  float scale;          // c
  float ratio, ratio2;  // c / scale as a sum
  DecodeArgs d;  // rows, max_length, waits
};

// A block's entry and what its keys [first, first + keys) have to do with it.
struct Entry {
  int64_t q0;
  int lq, row, end, p0;  // query rows; table row; keys that count; place of the first query
  bool seen, report;     // some row may see some key; the sequence is named twice
};
// First row of entry i, and one behind its last.
__device__ __forceinline__ int2 rows_of(const WeightsArgs &a, int i) {
  const int q0 = (int)min((int64_t)max(a.offsets[i], 0), a.tokens);
  return make_int2(q0, max(q0, (int)min((int64_t)a.offsets[i + 1], a.tokens)));
}
// also(row) runs beside the loads, for a row of the table.
template <typename Also>
__device__ __forceinline__ Entry open_entry(const WeightsArgs &a, const KvView &c, int first, int keys, int threads,
                                            Also also) {
  Entry e;
  const int i = blockIdx.y;
  const int2 rows = rows_of(a, i);
  e.row = a.d.sequences ? a.d.sequences[i] : i;
  int twice = 0;
  if (a.d.sequences)
    for (int j = threadIdx.x; j < i; j += threads)  // entries without rows take nobody's place
      if (a.d.sequences[j] == e.row) {
        const int2 others = rows_of(a, j);
        twice |= others.y > others.x;
      }
  int length = 0;
  if (e.row >= 0 && e.row < c.max_sequences) also(e.row);
  e.row = sequence_of(c, a.d, i, &length);
  e.q0 = rows.x;
  e.lq = rows.y - rows.x;
  e.end = (int)min((int64_t)length, a.weights_stride);
  e.p0 = length - e.lq;
  twice = __syncthreads_or(twice) && e.lq > 0;
  // within the first query's window, or a sink
  e.seen = e.lq > 0 && first < e.end && !twice &&
           (!a.window || first + keys > max(e.p0, 0) - (a.window - 1) || first < a.sinks);
  e.report = twice && first == 0 && length > 0;
  return e;
}

// ---------------------------------------------------------------------------
// On mma.sync tiles: for queries that no tensor map holds (broadcast ones) and groups of more than 64
// heads. Every block of 64 keys reads all of its entry's queries through shared memory; that and two
// blocks of four warps an SM bound it (last 128 queries of prompts of 3000 to 12000 tokens, 32 and 8
// heads of dim 128, 870 us, where the other kernel takes 69).
// ---------------------------------------------------------------------------

// The exponent's second term of a row, and the factor for what it leaves out. (A row without
// statistics gives nothing whatever its query holds, so its weights are not left to -infinity here:
// with a score that is not finite that is NaN.)
__device__ __forceinline__ void exponent_of(const WeightsArgs &a, float lse, float *z, float *factor) {
  const float hi = lse * a.ratio, lo = fmaf(lse, a.ratio2, fmaf(lse, a.ratio, -hi));
  *z = -hi;
  *factor = isfinite(hi) ? fmaf(lo, -kLn2, 1.0f) : 1.0f;
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(kThreads)
weights_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ WeightsArgs a,
               const __grid_constant__ KvView c) {
  using C = Cfg<DP>;
  constexpr unsigned kAll = 0xffffffffu;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[kWarps][C::kStages];
  __shared__ alignas(8) float lse_of[2][C::kTiles * kTileRows];
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
  const int group = a.group, dim = c.head_dim;
  const int first = blockIdx.x / ranks * kKeys, key = first + warp * kWarpKeys;
  const Entry e = open_entry(a, c, first, kKeys, kThreads, [](int) {});
  if (e.report && rank == 0 && tid == 0) atomicOr(c.status, DM_KV_BAD_SEQUENCE);
  if (!e.seen) return;  // all ranks alike
  const int64_t q0 = e.q0;
  const int lq = e.lq, row = e.row, end = e.end, p0 = e.p0;
  if (ranks > 1) cluster.sync();  // the others' shared memory is there

  // ---- tiles of query rows, of all key/value heads one after the other; this block's share
  const int rows = lq * group;  // a tile more is still below 2^31 by the call's check
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
      float z[2], factor[2], w[4];
      exponent_of(a, lse.x, &z[0], &factor[0]);
      exponent_of(a, lse.y, &z[1], &factor[1]);
#pragma unroll
      for (int i = 0; i < 4; i++)
        w[i] = (i & 1 ? lse.y : lse.x) == -INFINITY ? 0.0f : exp2_fast(fmaf(s[i] + s2[i], a.scale, z[i & 1])) * factor[i & 1];
      // some key is hidden from some row
      if (key + kWarpKeys - 1 > from || (a.window && to - key >= a.window && key + kWarpKeys > a.sinks)) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int r = tile * kTileRows + (lane & 3) * 2 + (i & 1);
          const int p = r < rows ? p0 + r / group : -1, j = key + (lane >> 2) + (i >> 1) * 8;
          const int last_place = a.window && j >= a.sinks ? (int)min((int64_t)j + a.window - 1, (int64_t)INT32_MAX) : INT32_MAX;
          w[i] = p >= j && p <= last_place ? w[i] : 0.0f;
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


// ---------------------------------------------------------------------------
// The same on tcgen05 tiles: 128 keys of one head are the rows of a product (TMEM lanes), COLS query
// rows its columns; with many query rows a block has twice 128 keys, which share the query tiles (all
// blocks together read the queries once for each of their key ranges, and that is what L2 has to
// give). A thread has one key: it reads its row of the product, weighs and sums it along
// the columns, and keeps the sum over all of the block's queries and heads. One warp each loads keys
// (in slabs of 64 values) and queries, issues products and fetches statistics.
//
// Bound, with many query rows, by the exponentials: a tile of 128 rows and 256 keys takes 2400 cycles,
// 2048 of them the exponential unit's (products of 128 columns and two halves: 64 columns took 1500
// for a quarter of that, most of it issue and waits); a block's first loads and its end cost 9000
// more, and a ragged batch does not fill the last round: last 128 queries of prompts of 3000 to 12000
// tokens 69 us, 39% of the exponential unit over all. With few rows by memory: one query of each of 16
// chats of 1186 to 3901 tokens, 32 and 8 heads of dim 128 (83 MB) 19 us, 4.3 TB/s, of which a block's
// chain of look-ups and the first keys' latency are a third. A quarter of the exponentials as a
// polynomial gained 7%, more lost; it is not here.
// ---------------------------------------------------------------------------

constexpr int kHalf = 128;  // keys of a product
constexpr int kMostSlabs = 12, kMostQueries = 6;
constexpr int kMostBuffers = 4;         // products in tensor memory
constexpr int kMostColumns = 128;
constexpr int kStatSlots = 8, kStatBatch = 4;  // tiles whose statistics are held, and are fetched at once

template <int DP, int COLS, int HALVES>
struct TileCfg {
  // Few query rows: blocks are short and mostly latency, so three share an SM.
  static constexpr int kBlocks = HALVES == 2 ? 1 : COLS <= 32 && DP <= 128 ? 3 : 2;
  static constexpr int kKeys = HALVES * kHalf;
  static constexpr int kSlab = kKeys * 128;  // bytes: 64 values of the keys
  // for rings, beside 8 (15 with 64 columns, 29 with 128) KB of the rest and 1 KB that a block costs
  static constexpr int kRoom = (kBlocks == 3 ? 66 : kBlocks == 1 ? 196 : COLS == 64 ? 97 : 104) * 1024;
  static constexpr int kQBytes = COLS * DP * 2;
  static constexpr int kSlabs = DP / 64;  // of a head
  // warps that weigh: with many query rows a second four, which take every other tile
  static constexpr int kGroups = COLS >= 64 ? 2 : 1, kSoft = 4 * kGroups * HALVES, kThreads = (kSoft + 4) * 32;
  // two heads' keys; with many query rows one and a half, and more query tiles
  static constexpr int kMay = (kRoom - 2 * kQBytes) / kSlab, kLike = COLS >= 64 ? (3 * kSlabs + 1) / 2 : 2 * kSlabs;
  static constexpr int kWant = kLike < kMay ? kLike : kMay;
  static constexpr int kKeySlots = kWant < kMostSlabs ? kWant : kMostSlabs;
  static constexpr int kLeft = (kRoom - kKeySlots * kSlab) / kQBytes;
  static constexpr int kQuerySlots = kLeft < kMostQueries ? kLeft : kMostQueries;
  static constexpr int kSmem = 1024 + kKeySlots * kSlab + kQuerySlots * kQBytes;
  static constexpr int kBuffers = HALVES * COLS > 128 ? 2 : 4, kTmem = kBuffers * HALVES * COLS;
  static_assert(kKeySlots >= kSlabs && kQuerySlots >= 2, "a head's keys and two query tiles fit");
};

template <int COLS>
struct TileSmem {
  static constexpr int kRowsOf = COLS < 32 ? 32 : COLS;  // a lane's at least
  uint64_t k_full[kMostSlabs], k_empty[kMostSlabs], q_full[kMostQueries], q_empty[kMostQueries];
  uint64_t z_full[kStatSlots], z_empty[kStatSlots], s_full[kMostBuffers], s_free[kMostBuffers], drain;
  alignas(16) float z[kStatSlots][kRowsOf], factor[kStatSlots][kRowsOf];  // of a tile's query rows
  alignas(16) int place[kStatSlots][kRowsOf];  // -1: no row, or one without statistics
  int holes[kStatSlots];                       // a row of the tile has no statistics
  uint32_t tmem;
  volatile int abort;
};

struct TileArgs {
  WeightsArgs w;
  int32_t tokens;  // of a query tile
  int32_t k_box;   // keys of a TMA box
};

__device__ __forceinline__ void arrive(uint64_t &bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&bar)) : "memory");
}
// Bounded wait of a warp that also ends when another role has given up.
__device__ __forceinline__ bool wait(volatile int &abort, int64_t limit, uint64_t &bar, uint32_t parity) {
  constexpr unsigned kAll = 0xffffffffu;
  const uint32_t b = smem_u32(&bar);
  if (__all_sync(kAll, mbar_look(b, parity))) return true;
  const long long start = clock64();
  while (!__all_sync(kAll, mbar_look(b, parity)))
    if (__any_sync(kAll, abort || clock64() - start > limit)) {
      abort = 1;
      return false;
    }
  return true;
}
template <int SLOTS>
struct Turn {  // a place in a ring
  int slot = 0;
  uint32_t round = 0;
  __device__ void next() {
    if (++slot == SLOTS) slot = 0, round++;
  }
  // What has been loaded lands before the block ends, whether or not somebody waits for it.
  __device__ void drain(uint64_t *full) {
    for (int n = min(SLOTS, (int)(round * SLOTS + slot)); n > 0; n--) {
      if (--slot < 0) slot = SLOTS - 1, round--;
      mbar_wait(smem_u32(&full[slot]), round & 1);
    }
  }
};
// Heads and query tiles of a block, one after the other.
struct Walk {
  int head, tile, first, behind, left;
  __device__ Walk(int u0, int u1, int t0, int t1)
      : head(u0 / (t1 - t0)), tile(t0 + u0 % (t1 - t0)), first(t0), behind(t1), left(u1 - u0) {}
  __device__ void next() {
    left--;
    if (++tile == behind) tile = first, head++;
  }
};

template <int DP, int COLS, int HALVES, bool BF16>
__global__ void __launch_bounds__((TileCfg<DP, COLS, HALVES>::kThreads), (TileCfg<DP, COLS, HALVES>::kBlocks))
tile_weights_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                    const __grid_constant__ TileArgs t, const __grid_constant__ KvView c) {
  using Cfg = TileCfg<DP, COLS, HALVES>;
  constexpr int kSoft = Cfg::kSoft, kGroups = Cfg::kGroups, kKeys = Cfg::kKeys, kSlab = Cfg::kSlab,
                kBuffers = Cfg::kBuffers;
  extern __shared__ uint8_t raw[];
  __shared__ TileSmem<COLS> sh;
  __shared__ float sums[kMostRanks * kGroups][kKeys];
  const WeightsArgs &a = t.w;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = (smem_u32(raw) + 1023) & ~1023u, q_ring = base + Cfg::kKeySlots * kSlab;
  auto cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map));
    asm volatile("prefetch.tensormap [%0];" ::"l"(&q_map));
  }
  if (tid < kMostSlabs) mbar_init(smem_u32(&sh.k_full[tid]), 1), mbar_init(smem_u32(&sh.k_empty[tid]), 1);
  if (tid < kMostQueries) mbar_init(smem_u32(&sh.q_full[tid]), 1), mbar_init(smem_u32(&sh.q_empty[tid]), 1);
  if (tid < kStatSlots) mbar_init(smem_u32(&sh.z_full[tid]), 1), mbar_init(smem_u32(&sh.z_empty[tid]), 4 * HALVES);
  if (tid < kBuffers) mbar_init(smem_u32(&sh.s_full[tid]), 1), mbar_init(smem_u32(&sh.s_free[tid]), 4 * HALVES);
  if (tid == 0) {
    sh.abort = 0;
    mbar_init(smem_u32(&sh.drain), 1);
  }
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  wait_for_previous();
  let_next_start();
  const int first = blockIdx.x / ranks * kKeys;
  int page = 0;  // of the loading warp's lane: its box
  const Entry e = open_entry(a, c, first, kKeys, Cfg::kThreads, [&](int row) {
    const int key = first + lane * t.k_box;
    if (warp == kSoft && lane * t.k_box < kKeys && key / c.page_tokens < c.max_pages)
      page = c.table[(int64_t)row * c.max_pages + key / c.page_tokens];
  });
  if (e.report && rank == 0 && tid == 0) atomicOr(c.status, DM_KV_BAD_SEQUENCE);
  if (!e.seen) return;  // all ranks alike
  // query tiles that see some of the keys
  const int per = t.tokens, tiles = (e.lq + per - 1) / per;
  const int t0 = max(0, first - e.p0) / per;
  int t1 = tiles;
  if (a.window && first >= a.sinks) {  // the last row whose window reaches the last key
    const int64_t last = (int64_t)first + kKeys - 2 + a.window - e.p0;
    if (last < e.lq) t1 = last < 0 ? 0 : (int)(last / per) + 1;
  }
  if (t1 <= t0) return;
  // Loads begin at once. Tensor memory is for the warps that weigh and the one of the products; the
  // others' shared memory (the barrier's other half) is needed at the end.
  if (ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  constexpr int kProducts = kSoft + 2;
  if (warp < kSoft || warp == kProducts) {
    if (warp == kProducts) tmem_alloc(smem_u32(&sh.tmem), Cfg::kTmem);
    fence_before();
    asm volatile("bar.sync 1, %0;" ::"n"((kSoft + 1) * 32) : "memory");
    fence_after();
  }
  const uint32_t tmem = *(volatile uint32_t *)&sh.tmem;
  const bool adds = rank == 0 && tid < kKeys && first + tid < e.end;
  const float old = adds ? a.weights[e.row * a.weights_stride + first + tid] : 0.0f;

  // this block's share of heads x tiles
  const int64_t all = (int64_t)(t1 - t0) * c.kv_heads;
  const int u0 = (int)(all * rank / ranks), u1 = (int)(all * (rank + 1) / ranks);
  const int group = a.group;
  const int64_t limit = a.d.wait_limit;
  float total = 0.0f;
  bool ok = true;
  Walk at(u0, u1, t0, t1);

  if (warp >= kSoft) {
    const bool lead = lane == 0;
    if (warp == kSoft) {
      // ---- keys: boxes of one page each, a lane for each
      const int used = (min(kKeys, e.end - first) + t.k_box - 1) / t.k_box;
      const int place = (first + lane * t.k_box) & (c.page_tokens - 1);
      Turn<Cfg::kKeySlots> k;
      const int behind = u1 > u0 ? (u1 - 1) / (t1 - t0) + 1 : 0;
      for (int h = at.head; h < behind && ok; h++)
        for (int slab = 0; slab < Cfg::kSlabs; slab++, k.next()) {
          if (k.round > 0 && !(ok = wait(sh.abort, limit, sh.k_empty[k.slot], (k.round - 1) & 1))) break;
          const uint32_t bar = smem_u32(&sh.k_full[k.slot]);
          if (lead) mbar_expect_tx(bar, used * t.k_box * 128);
          __syncwarp();
          if (lane < used)
            tma_load_4d(base + k.slot * kSlab + lane * t.k_box * 128, &k_map, slab * 64, place, h, page, bar);
        }
      if (rank == 0 && lane < used && (unsigned)page >= (unsigned)c.pages) atomicOr(c.status, DM_KV_BAD_TOKEN);
      k.drain(sh.k_full);
    } else if (warp == kSoft + 1) {
      // ---- queries
      Turn<Cfg::kQuerySlots> q;
      for (; at.left > 0; at.next(), q.next()) {
        if (q.round > 0 && !(ok = wait(sh.abort, limit, sh.q_empty[q.slot], (q.round - 1) & 1))) break;
        const uint32_t bar = smem_u32(&sh.q_full[q.slot]);
        if (lead) mbar_expect_tx(bar, Cfg::kSlabs * per * group * 128);
        __syncwarp();
        if (lane < Cfg::kSlabs)
          tma_load_4d(q_ring + q.slot * Cfg::kQBytes + lane * COLS * 128, &q_map, lane * 64, 0, at.head,
                      (int)(e.q0 + (int64_t)at.tile * per), bar);
      }
      q.drain(sh.q_full);
    } else if (warp == kSoft + 2) {
      // ---- products
      constexpr uint32_t kIdesc = (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)(COLS >> 3) << 17) |
                                  ((uint32_t)(128 >> 4) << 24);
      Turn<Cfg::kKeySlots> k;
      Turn<Cfg::kQuerySlots> q;
      Turn<kBuffers> s;
      const uint32_t one = elect_one(), out = uniform(tmem);
      bool fresh = true;  // a head's first tile
      for (; at.left > 0; at.next(), q.next(), s.next()) {
        if (!(ok = wait(sh.abort, limit, sh.q_full[q.slot], q.round & 1))) break;
        if (s.round > 0 && !(ok = wait(sh.abort, limit, sh.s_free[s.slot], (s.round - 1) & 1))) break;
        const bool ends = at.left == 1 || at.tile + 1 == at.behind;
        Turn<Cfg::kKeySlots> slab = k;
#pragma unroll
        for (int i = 0; i < Cfg::kSlabs; i++, slab.next()) {
          if (fresh && !(ok = wait(sh.abort, limit, sh.k_full[slab.slot], slab.round & 1))) break;
          fence_after();
          const uint64_t kd = sw128_desc(base + slab.slot * kSlab);
          const uint64_t qd = sw128_desc(q_ring + q.slot * Cfg::kQBytes + i * COLS * 128);
#pragma unroll
          for (int half = 0; half < HALVES; half++)
#pragma unroll
            for (int j = 0; j < 4; j++)
              mma_ss_if(one, out + (s.slot * HALVES + half) * COLS, kd + (half * kHalf * 128 >> 4) + j * 2, qd + j * 2,
                        kIdesc, i > 0 || j > 0);
          if (ends) commit_if(one, smem_u32(&sh.k_empty[slab.slot]));
        }
        if (!ok) break;
        commit_if(one, smem_u32(&sh.s_full[s.slot]));
        commit_if(one, smem_u32(&sh.q_empty[q.slot]));
        fresh = ends;
        if (ends) k = slab;
      }
      // products in flight end before tensor memory is let go, whoever has given up
      commit_if(one, smem_u32(&sh.drain));
      mbar_wait(smem_u32(&sh.drain), 0);
    } else {
      // ---- statistics: a lane's rows of several tiles at once, a batch ahead
      constexpr int kRowsOf = (COLS + 31) / 32;
      int token[kRowsOf], head[kRowsOf];
#pragma unroll
      for (int k = 0; k < kRowsOf; k++) {
        const int r = lane + k * 32;
        token[k] = r < per * group ? r / group : INT32_MAX / 2;
        head[k] = r % group;
      }
      float lse[kStatBatch][kRowsOf];
      Walk ahead = at;
      auto fetch = [&]() {
#pragma unroll
        for (int b = 0; b < kStatBatch; b++, ahead.next())
#pragma unroll
          for (int k = 0; k < kRowsOf; k++) {
            const int64_t i = (int64_t)ahead.tile * per + token[k];
            lse[b][k] = ahead.left > 0 && i < e.lq ? a.lse[(e.q0 + i) * a.heads + ahead.head * group + head[k]] : -INFINITY;
          }
      };
      fetch();
      Turn<kStatSlots> s;
      while (at.left > 0 && ok) {
        float z[kStatBatch][kRowsOf], factor[kStatBatch][kRowsOf];
        bool none[kStatBatch][kRowsOf];
#pragma unroll
        for (int b = 0; b < kStatBatch; b++)
#pragma unroll
          for (int k = 0; k < kRowsOf; k++) {
            exponent_of(a, lse[b][k], &z[b][k], &factor[b][k]);
            none[b][k] = lse[b][k] == -INFINITY;
          }
        fetch();
#pragma unroll
        for (int b = 0; b < kStatBatch; b++) {
          if (at.left <= 0) break;
          if (s.round > 0 && !(ok = wait(sh.abort, limit, sh.z_empty[s.slot], (s.round - 1) & 1))) break;
          bool hole = false;
#pragma unroll
          for (int k = 0; k < kRowsOf; k++) {
            const int64_t i = (int64_t)at.tile * per + token[k];
            sh.z[s.slot][lane + k * 32] = z[b][k];
            sh.factor[s.slot][lane + k * 32] = factor[b][k];
            sh.place[s.slot][lane + k * 32] = i < e.lq && !none[b][k] ? e.p0 + (int)i : -1;
            hole |= i < e.lq && none[b][k];
          }
          hole = __any_sync(0xffffffffu, hole);
          if (lead) sh.holes[s.slot] = hole;
          __syncwarp();
          if (lead) arrive(sh.z_full[s.slot]);
          at.next(), s.next();
        }
      }
    }
  } else {
    // ---- weights: one key a thread
    const int half = (warp >> 2) % HALVES, mine = (warp >> 2) / HALVES;
    const int near = first + half * kHalf, far = near + kHalf - 1, key = near + (tid & (kHalf - 1));
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const uint64_t cc = pair(a.scale, a.scale);
    // the key is seen from its own place to this one
    const int last_place = a.window && key >= a.sinks ? (int)min((int64_t)key + a.window - 1, (int64_t)INT32_MAX) : INT32_MAX;
    Turn<kBuffers> s;
    Turn<kStatSlots> z;
    for (int turn = 0; at.left > 0; at.next(), s.next(), z.next(), turn ^= kGroups - 1) {
      if (turn != mine) continue;
      if (!(ok = wait(sh.abort, limit, sh.z_full[z.slot], z.round & 1))) break;
      if (!(ok = wait(sh.abort, limit, sh.s_full[s.slot], s.round & 1))) break;
      fence_after();
      const int from = e.p0 + at.tile * per, count = min(per, e.lq - at.tile * per), to = from + count - 1;
      // every key is seen by every row, all have statistics, and there are as many as columns
      const bool clear = count * group == COLS && far <= from &&
                         (!a.window || to - near < a.window || far < a.sinks) && !sh.holes[z.slot];
      constexpr int kStep = COLS < 32 ? COLS : 32;
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int j0 = 0; j0 < COLS; j0 += kStep) {
        float x[kStep];
#pragma unroll
        for (int j = 0; j < kStep; j += 16)
          tmem_ld16(tmem + lanes + (s.slot * HALVES + half) * COLS + j0 + j, reinterpret_cast<uint32_t *>(x + j));
        tmem_wait_ld();
        if (j0 + kStep == COLS) {
          fence_before();
          __syncwarp();
          if (lane == 0) arrive(sh.s_free[s.slot]);
        }
#pragma unroll
        for (int j = 0; j < kStep; j += 4) {
          const float4 y = *reinterpret_cast<const float4 *>(&sh.z[z.slot][j0 + j]);
          const uint64_t y0 = fma2(pair(x[j], x[j + 1]), cc, pair(y.x, y.y));
          const uint64_t y1 = fma2(pair(x[j + 2], x[j + 3]), cc, pair(y.z, y.w));
          x[j] = exp2_fast(__uint_as_float((uint32_t)y0)), x[j + 1] = exp2_fast(__uint_as_float((uint32_t)(y0 >> 32)));
          x[j + 2] = exp2_fast(__uint_as_float((uint32_t)y1)), x[j + 3] = exp2_fast(__uint_as_float((uint32_t)(y1 >> 32)));
        }
        if (!clear) {
#pragma unroll
          for (int j = 0; j < kStep; j += 4) {
            const int4 p = *reinterpret_cast<const int4 *>(&sh.place[z.slot][j0 + j]);
            x[j] = p.x >= key && p.x <= last_place ? x[j] : 0.0f;
            x[j + 1] = p.y >= key && p.y <= last_place ? x[j + 1] : 0.0f;
            x[j + 2] = p.z >= key && p.z <= last_place ? x[j + 2] : 0.0f;
            x[j + 3] = p.w >= key && p.w <= last_place ? x[j + 3] : 0.0f;
          }
        }
#pragma unroll
        for (int j = 0; j < kStep; j += 4) {
          const float4 f = *reinterpret_cast<const float4 *>(&sh.factor[z.slot][j0 + j]);
          sum[0] = fma2(pair(x[j], x[j + 1]), pair(f.x, f.y), sum[0]);
          sum[1] = fma2(pair(x[j + 2], x[j + 3]), pair(f.z, f.w), sum[1]);
        }
      }
      __syncwarp();
      if (lane == 0) arrive(sh.z_empty[z.slot]);
      sum[0] = add2(sum[0], sum[1]);
      total += __uint_as_float((uint32_t)sum[0]) + __uint_as_float((uint32_t)(sum[0] >> 32));
    }
  }
  fence_before();
  __syncthreads();
  if (tid == 0 && sh.abort) atomicExch(a.d.timeout, 1);
  if (warp == kProducts) {
    fence_after();
    tmem_dealloc(tmem, Cfg::kTmem);
  }
  // ---- the sums of the ranks, and of the two groups of each, in order
  if (ranks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (ranks * kGroups > 1) {
    if (warp < kSoft) {
      float *there = ranks > 1 ? cluster.map_shared_rank(&sums[0][0], 0) : &sums[0][0];
      there[(rank * kGroups + tid / kKeys) * kKeys + tid % kKeys] = total;
    }
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    if (!adds) return;
    total = 0.0f;
    for (int i = 0; i < ranks * kGroups; i++) total += sums[i][tid];
  }
  if (adds) a.weights[e.row * a.weights_stride + first + tid] = old + total;
}

template <int DP, int COLS, int HALVES>
int32_t launch_tiles(bool bf16, dim3 grid, int ranks, const CUtensorMap *maps, const TileArgs &t, const KvView &c,
                     cudaStream_t s) {
  using Cfg = TileCfg<DP, COLS, HALVES>;
  auto fn = bf16 ? tile_weights_kernel<DP, COLS, HALVES, true> : tile_weights_kernel<DP, COLS, HALVES, false>;
  DM_CUDA(dm::ensure_smem_limit((const void *)fn), "attention shared memory");
  return launch_clusters("weights launch", fn, grid, ranks, Cfg::kThreads, Cfg::kSmem, s, maps[0], maps[1], t, c);
}
template <int DP>
int32_t launch_tiles(bool bf16, int columns, dim3 grid, int ranks, const CUtensorMap *maps, const TileArgs &t,
                     const KvView &c, cudaStream_t s) {
  if (columns == 16) return launch_tiles<DP, 16, 1>(bf16, grid, ranks, maps, t, c, s);
  if (columns == 32) return launch_tiles<DP, 32, 1>(bf16, grid, ranks, maps, t, c, s);
  if constexpr (DP == 256) return launch_tiles<DP, 64, 2>(bf16, grid, ranks, maps, t, c, s);
  else
    return columns == 64 ? launch_tiles<DP, 64, 1>(bf16, grid, ranks, maps, t, c, s)
                         : launch_tiles<DP, 128, 2>(bf16, grid, ranks, maps, t, c, s);
}

template <int DP, bool BF16>
int32_t launch_weights(dim3 grid, int ranks, const CUtensorMap &map, const WeightsArgs &a, const KvView &c,
                       cudaStream_t s) {
  auto fn = weights_kernel<DP, BF16>;
  DM_CUDA(dm::ensure_smem_limit((const void *)fn), "attention shared memory");
  return launch_clusters("weights launch", fn, grid, ranks, kThreads, Cfg<DP>::kSmem, s, map, a, c);
}

constexpr int kSms = 148;

// c and c / scale. Scores are the tensor cores' sums as they are, which cut a partial sum off where the
// next 16 products are added to it: they come out small by up to 1.2 times 2^-26 of themselves a step
// (f16: 2.4), and products that leave nothing to cut off are exact. Attention's own statistics are made
// from such scores, too, so with them a row's weights come to one: 160 rows with scores of 8 times
// normal, dim 64 to 256, to 2 10^-6 (a scale that gives the cut back on average 1 to 9 10^-6, and exact
// products up to 1.5 10^-5 too large, though with a lse from exact scores sums are 2 to 4 times nearer).
void set_scale(WeightsArgs *a, double scale) {
  a->scale = (float)(scale * 1.4426950408889634);
  a->ratio = (float)(a->scale / scale);
  a->ratio2 = (float)(a->scale / scale - a->ratio);
}

// How many blocks share the queries of their keys. Microseconds on one B200, as measured: a block
// has 6 besides (8 in a cluster) its keys at its part of an SM's 44 KB each, or its query tiles:
// 1.8 for 128 rows and 256 keys, 0.8 for 64 and 128, 0.4 and 0.3 for 32 and 16.
int tile_ranks(int64_t blocks, int at_once, int keys, int dim, int kv_heads, int columns, int tiles) {
  const float tile = columns == 128 || keys > kHalf ? 1.8f : columns == 64 ? 0.8f : columns == 32 ? 0.4f : 0.3f;
  int best = 1;
  float best_us = 0.0f;
  for (int ranks = 1; ranks <= kMostRanks && ranks <= kv_heads * tiles; ranks *= 2) {
    const float share = std::min((float)at_once, std::max(1.0f, (float)blocks * ranks / kSms));
    const float work = kv_heads * std::max(keys * dim * 2 / 44000.0f * share, tiles * tile) / ranks;
    const int64_t rounds = (blocks * ranks + (int64_t)kSms * at_once - 1) / ((int64_t)kSms * at_once);
    const float us = rounds * ((ranks > 1 ? 8.0f : 6.0f) + work);
    if (ranks == 1 || us < best_us) best = ranks, best_us = us;
  }
  return best;
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
  // the rows of a head are counted in 32 bits up to a whole tile
  if (in->tokens * in->heads > INT32_MAX - kTileRows) return fail(DM_ERR_OVERFLOW, "too many query rows");
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
  set_scale(&a, in->scale == 0.0f ? 1.0 / std::sqrt((double)d.head_dim) : in->scale);
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
  cudaStream_t s = (cudaStream_t)stream;
  const bool bf = d.type == DM_BF16;
  const int64_t busy = std::min<int64_t>(in->sequences, in->tokens), each = (in->tokens + busy - 1) / busy;
  CUtensorMap maps[2];
  if (tile_queries_fit(a.q_stride, a.group) && a.group <= 64) {
    int columns = d.head_dim > 128 ? 64 : kMostColumns;
    while (columns > 16 && columns / 2 >= each * a.group) columns /= 2;
    TileArgs t{};
    t.w = a;
    t.tokens = columns / a.group;
    t.k_box = std::min<int>(d.page_tokens, kHalf);
    if (!describe_queries(d.type, in->q, a.q_stride, d.head_dim, a.group, d.kv_heads, in->tokens, t.tokens, &maps[0]) ||
        !describe_keys(d.type, cache->view, in->layer, t.k_box, &maps[1]))
      return fail(DM_ERR_COMMAND, "could not describe the attention tensors for TMA");
    const int per_block = columns == kMostColumns || (columns == 64 && d.head_dim > 128) ? 2 * kHalf : kHalf;
    const int64_t blocks = (keys + per_block - 1) / per_block;
    const int at_once = per_block > kHalf ? 1 : columns <= 32 && d.head_dim <= 128 ? 3 : 2;
    const int ranks = tile_ranks(blocks * in->sequences, at_once, per_block, d.head_dim, d.kv_heads, columns,
                                 (int)((each + t.tokens - 1) / t.tokens));
    const dim3 grid((unsigned)(blocks * ranks), in->sequences);
    return d.head_dim <= 64    ? launch_tiles<64>(bf, columns, grid, ranks, maps, t, cache->view, s)
           : d.head_dim <= 128 ? launch_tiles<128>(bf, columns, grid, ranks, maps, t, cache->view, s)
                               : launch_tiles<256>(bf, columns, grid, ranks, maps, t, cache->view, s);
  }
  if (!describe_chunks(d.type, cache->view, in->layer, kWarpKeys, maps))
    return fail(DM_ERR_COMMAND, "could not describe the cache for TMA");
  const int64_t tiles = (keys + kKeys - 1) / kKeys;
  // few blocks: several share the queries of their keys
  const int64_t steps = (each * a.group + kTileRows - 1) / kTileRows * d.kv_heads;
  int ranks = 1;
  while (ranks < kMostRanks && tiles * in->sequences * ranks < 2 * kSms && steps >= 2 * ranks) ranks *= 2;
  const dim3 grid((unsigned)(tiles * ranks), in->sequences);
  if (d.head_dim <= 64)
    return bf ? launch_weights<64, true>(grid, ranks, maps[0], a, cache->view, s)
              : launch_weights<64, false>(grid, ranks, maps[0], a, cache->view, s);
  if (d.head_dim <= 128)
    return bf ? launch_weights<128, true>(grid, ranks, maps[0], a, cache->view, s)
              : launch_weights<128, false>(grid, ranks, maps[0], a, cache->view, s);
  return bf ? launch_weights<256, true>(grid, ranks, maps[0], a, cache->view, s)
            : launch_weights<256, false>(grid, ranks, maps[0], a, cache->view, s);
}
