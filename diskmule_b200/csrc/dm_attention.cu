// dm_attention.cu -- attention: argument checks, launches, and the kernels on mma.sync tiles
// of 16 query rows.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "dm_attention.cuh"
#include "dm_attention_tc.cuh"
#include "dm_mma.cuh"
#include "dm_tcgen05.cuh"

using dmi::fail;

namespace dma {

using namespace dm::tc;

// ---------------------------------------------------------------------------
// 16 query rows against a range of keys. The block's warps take chunks of 16 keys in turn,
// each with its own ring of shared-memory stages and its own softmax state, so nothing in the
// loop waits for another warp; their states join at the end. Chunks of a cache come by TMA
// (rows of 64 values, 128-byte swizzle; a few instructions of one lane, where cp.async took a
// third of the loop's), those of a prompt by cp.async into the same layout.
//
// Bound by memory where there is enough to read: 64 sequences of 1500 own tokens, 8 key/value
// heads of dim 128, 67 us, 5.9 TB/s; 256 of them 236 us, 6.7. Small calls are latency (table,
// queries, keys, join of the warps): 2 sequences of 200 tokens 5 us. Weights are rounded to 16
// bits before the product (its operands have one type), the sums are not. Prompts whose tensors
// are broadcast (a stride of zero) take this kernel, too, and chunks of few query rows: one token
// over 98304 (32 and 8 heads of dim 128, 403 MB) 66 us besides the join's 6, 6.1 TB/s.
// ---------------------------------------------------------------------------

constexpr int kRows = 16;    // query rows of a block: one mma tile
constexpr int kChunk = 16;   // keys of a step of one warp; pages are multiples of it
constexpr int kStages = 3;   // of a warp's ring
constexpr int kJoinThreads = 128;
constexpr int kMostJoined = 8;     // shared parts that a block of the own part joins itself
constexpr int kMostParts = 512;

enum Mode { kPrompt, kOwn, kShared, kChunks };

template <int DP, int WARPS>
struct RowsCfg {
  static constexpr int kThreads = WARPS * 32;
  static constexpr int kTile = kChunk * DP * 2;   // bytes of a K or V tile
  static constexpr int kSlab = kChunk * 128;      // 64 values of its rows
  static constexpr int kRing = kStages * 2 * kTile;
  static constexpr int kJoin = WARPS * kRows * DP * 4;
  // room for the warps' states, too; rings are aligned to 1024 bytes
  static constexpr int kSmem = 1024 + WARPS * kRing;
  static_assert(kJoin <= WARPS * kRing, "the states fit the rings");
  static constexpr int kBlocks = kSmem <= 112 * 1024 ? 2 : 1;  // per SM
};

// Add a state (ml, o) to the sums that refer to z.
__device__ __forceinline__ void add_state(float &l, float4 &v, float2 ml, float4 o, float z) {
  const float f = exp2_fast(ml.x - z);
  l += ml.y * f;
  v.x += o.x * f, v.y += o.y * f, v.z += o.z * f, v.w += o.w * f;
}

template <int WARPS>
struct RowsSmem {
  int64_t q[kRows];     // element offset of the row's query, -1: no row
  int64_t out[kRows];   // element offset of its output
  int64_t index[kRows]; // its row in lse and in the parts
  int low[kRows], high[kRows];  // the keys that it sees
  int table[kRows];             // its sequence's row of the page table
  float2 ml[WARPS][kRows];
  uint64_t full[WARPS][kStages];  // a chunk of a warp has landed
  TileOf tile;
};

template <int MODE, int DP, int WARPS, bool BF16>
__global__ void __launch_bounds__(WARPS * 32, (RowsCfg<DP, WARPS>::kBlocks))
rows_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
            const __grid_constant__ PromptArgs p, const __grid_constant__ DecodeArgs d,
            const __grid_constant__ KvView c) {
  using Cfg = RowsCfg<DP, WARPS>;
  constexpr int kWarps = WARPS, kThreads = Cfg::kThreads;
  constexpr bool kPacked = MODE == kPrompt || MODE == kChunks;  // query rows by offsets
  extern __shared__ uint8_t raw[];
  uint8_t *smem = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
  __shared__ RowsSmem<WARPS> sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (MODE != kPrompt && tid < WARPS * kStages) mbar_init(smem_u32(&sh.full[tid / kStages][tid % kStages]), 1);
  if (MODE != kPrompt) asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  const int dim = MODE == kPrompt ? p.dim : c.head_dim;
  const int group = kPacked ? p.group : d.group;

  // The own part of a decode call reads nothing that the shared part's kernel before it
  // writes, and that one has waited for what both read: they run side by side.
  const bool beside = MODE == kOwn && d.first_part > 0;
  if (!beside) wait_for_previous();
  let_next_start();

  // ---- the block's rows, its keys and where they lie
  int kv_head, first = 0, last, table_row = 0;
  int64_t k0 = 0;  // prompt: first key row
  if (kPacked) {
    kv_head = MODE == kPrompt ? blockIdx.y : blockIdx.x % c.kv_heads;
    if (warp == 0) {
      const TileOf t = MODE == kPrompt ? find_tile(p, group, kRows, blockIdx.x)
                                       : find_sparse_tile(p, group, kRows, blockIdx.x / c.kv_heads);
      if (lane == 0) sh.tile = t;
    }
    __syncthreads();
    const TileOf t = sh.tile;
    if (t.seq < 0) return;
    k0 = t.k0;
    const int lq = t.q1 - t.q0;
    int lk = t.k1 - t.k0;
    if (MODE == kChunks) table_row = sequence_of(c, d, t.seq, &lk);
    if (tid < kRows) {
      const int64_t r = (int64_t)t.tile * kRows + tid;
      const int token = (int)(r / group), head = kv_head * group + (int)(r % group);
      const int64_t at = t.q0 + token;
      const bool valid = token < lq;
      sh.q[tid] = valid ? at * p.q_stride[0] + head * p.q_stride[1] : -1;
      sh.out[tid] = at * p.out_stride[0] + head * p.out_stride[1];
      sh.index[tid] = at * p.heads + head;
      sh.low[tid] = low_of(p, lq, lk, token);
      sh.high[tid] = high_of(p, lq, lk, token);
    }
  } else {
    const int rows = MODE == kOwn ? group : d.batch * group;
    const int blocks = (rows + kRows - 1) / kRows;
    const int rb = blockIdx.x % blocks;
    kv_head = (blockIdx.x / blocks) % c.kv_heads;
    const int entry = MODE == kOwn ? blockIdx.x / blocks / c.kv_heads : 0;
    if (tid < kRows) {
      const int r = rb * kRows + tid;
      const int b = MODE == kOwn ? entry : r / group;
      const int head = kv_head * group + r % group;
      const bool valid = r < rows;
      int length = 0;
      sh.table[tid] = valid ? sequence_of(c, d, b, &length) : 0;
      sh.q[tid] = valid ? b * d.q_stride[0] + head * d.q_stride[1] : -1;
      sh.out[tid] = b * d.out_stride[0] + head * d.out_stride[1];
      sh.index[tid] = (int64_t)b * d.heads + head;
      const int low = d.window ? max(0, length - d.window) : 0;
      sh.low[tid] = MODE == kOwn ? max(low, d.shared) : low;
      sh.high[tid] = MODE == kOwn ? length : min(length, d.shared);
    }
  }
  __syncthreads();
  int low = INT32_MAX, high = 0;
  // Pages are looked up for the row that sees the most keys: the others, which may be shorter
  // or empty, have the same pages as far as they reach and no entries behind that.
#pragma unroll
  for (int r = 0; r < kRows; r++)
    if (sh.q[r] >= 0) {
      if (!kPacked && sh.high[r] > high) table_row = sh.table[r];
      low = min(low, sh.low[r]), high = max(high, sh.high[r]);
    }
  low = low / kChunk * kChunk;
  Range range{};  // chunks: keys go by their number among those that are seen
  if (MODE == kChunks) {
    range = range_of(p, low, high, kChunk);
    low = 0, high = range.keys;
  }
  first = low, last = high;
  if (MODE != kPrompt && high > low) {
    // this block's part: whole chunks for every warp, and no fewer than 128 keys
    const int per = max(128, (((high - low) + d.splits - 1) / d.splits + 63) / 64 * 64);
    first = (int)min((int64_t)high, low + (int64_t)blockIdx.y * per);
    last = (int)min((int64_t)high, (int64_t)first + per);
  }

  // ---- this thread's rows (tid % 32 / 4 and + 8) and its query fragments
  const int ra = lane >> 2, rb8 = ra + 8;
  const int64_t qa = sh.q[ra], qb = sh.q[rb8];
  // a row that is not there sees everything: its results are dropped
  const int low_a = qa < 0 ? 0 : sh.low[ra], high_a = qa < 0 ? INT32_MAX : sh.high[ra];
  const int low_b = qb < 0 ? 0 : sh.low[rb8], high_b = qb < 0 ? INT32_MAX : sh.high[rb8];
  const uint16_t *qp = kPacked ? p.q : d.q;
  uint32_t qf[DP / 16][4];
#pragma unroll
  for (int k = 0; k < DP / 16; k++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int col = k * 16 + h * 8 + (lane & 3) * 2;
      const bool in = col < dim;
      qf[k][h * 2] = in && qa >= 0 ? *reinterpret_cast<const uint32_t *>(qp + qa + col) : 0u;
      qf[k][h * 2 + 1] = in && qb >= 0 ? *reinterpret_cast<const uint32_t *>(qp + qb + col) : 0u;
    }

  // ---- the warp's ring: V behind K, slabs of 64 values, 128-byte swizzle
  const uint32_t ring = smem_u32(smem) + warp * Cfg::kRing;
  constexpr int kVec = DP / 8;  // 16-byte vectors of a row
  auto at = [](int r, int v) { return (uint32_t)((v >> 3) * Cfg::kSlab + r * 128 + ((v ^ r) & 7) * 16); };
  const int page_bits = MODE == kPrompt ? 0 : 31 - __clz(c.page_tokens);  // pages are powers of two
  // As the table has it: a number outside the pool is outside the map, too, and reads as zeros.
  // It is looked at when it is used, so that nothing waits for it here, and reported at the end.
  uint32_t largest = 0;
  auto key_of = [&](int number) -> int { return MODE == kChunks ? range.key(number) : number; };
  auto page_of = [&](int key) -> int {
    return MODE == kPrompt || key >= last ? -1 : c.table[(int64_t)table_row * c.max_pages + (key_of(key) >> page_bits)];
  };
  auto load = [&](int key, int page, int stage) {
    const uint32_t kd = ring + stage * 2 * Cfg::kTile, vd = kd + Cfg::kTile;
    if (MODE == kPrompt) {
      const uint16_t *kb = p.k + (k0 + key) * p.k_stride[0] + kv_head * p.k_stride[1];
      const uint16_t *vb = p.v + (k0 + key) * p.v_stride[0] + kv_head * p.v_stride[1];
#pragma unroll
      for (int i = 0; i < kChunk * kVec / 32; i++) {
        const int n = i * 32 + lane, r = n / kVec, v = n % kVec;
        const bool valid = key + r < last && v < dim / 8;
        cp16(kd + at(r, v), valid ? kb + r * p.k_stride[0] + v * 8 : kb, valid);
        cp16(vd + at(r, v), valid ? vb + r * p.v_stride[0] + v * 8 : vb, valid);
      }
    } else {
      const uint32_t bar = smem_u32(&sh.full[warp][stage]);
      if (lane == 0) mbar_expect_tx(bar, 2 * Cfg::kTile);
      __syncwarp();
      largest = max(largest, (uint32_t)page);
      if (lane < 2 * (DP / 64)) {  // one slab each
        const bool is_v = lane >= DP / 64;
        const int slab = lane % (DP / 64);
        tma_load_4d((is_v ? vd : kd) + slab * Cfg::kSlab, is_v ? &v_map : &k_map, slab * 64,
                    key_of(key) & (c.page_tokens - 1), kv_head, page, bar);
      }
    }
  };

  float o[DP / 8][4];
#pragma unroll
  for (int i = 0; i < DP / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  float ma = -INFINITY, mb = -INFINITY, la = 0.0f, lb = 0.0f;
  const float scale = kPacked ? p.scale : d.scale;
  const int sinks = MODE == kChunks && p.window ? p.sinks : 0;
  constexpr float kRoom = kRowsHeadroom<BF16>;

  constexpr int kStep = kWarps * kChunk;
  int key_load = first + warp * kChunk;
  int page = page_of(key_load), page2 = page_of(key_load + kStep);
  auto issue = [&](int stage) {
    if (key_load < last) {
      const int next = page_of(key_load + 2 * kStep);  // two steps ahead of its use
      load(key_load, page, stage);
      page = page2, page2 = next;
    }
    key_load += kStep;
    if (MODE == kPrompt) asm volatile("cp.async.commit_group;");
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; s++) issue(s);
  int stage = 0;
  uint32_t parity = 0;  // of the ring's round
  for (int key = first + warp * kChunk; key < last; key += kStep) {
    if (MODE == kPrompt) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2));
    } else if (!__all_sync(0xffffffffu, copy_landed(smem_u32(&sh.full[warp][stage]), parity, d.wait_limit))) {
      // the copies in flight land before the block's states take their place
      if (lane == 0) atomicExch(d.timeout, 1);
      for (; key < min(key_load, last); key += kStep) {
        mbar_wait(smem_u32(&sh.full[warp][stage]), parity);
        if (++stage == kStages) stage = 0, parity ^= 1;
      }
      break;
    }
    __syncwarp();  // all lanes' copies are there, and all have left the stage that is next
    issue(stage == 0 ? kStages - 1 : stage - 1);
    const uint32_t kt = ring + stage * 2 * Cfg::kTile, vt = kt + Cfg::kTile;
    // two chains of products per 8 keys: one would be bound by the latency of its links
    float s[2][4] = {}, s2[2][4] = {};
    {
      const int r = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
      for (int k = 0; k < DP / 16; k++) {
        uint32_t b[4];
        const int v = 2 * k + ((lane >> 3) & 1);
        ldm4(kt + at(r, v), b);
        mma16816<BF16>(k & 1 ? s2[0] : s[0], qf[k], b[0], b[1]);
        mma16816<BF16>(k & 1 ? s2[1] : s[1], qf[k], b[2], b[3]);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) s[0][i] += s2[0][i], s[1][i] += s2[1][i];
    }
    // scores, masked, and the new maxima
    float na = ma, nb = mb;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int j = key_of(key) + t * 8 + (lane & 3) * 2 + e;
        const bool sink = MODE == kChunks && j < sinks;
        s[t][e] = (j >= low_a || sink) && j < high_a ? s[t][e] * scale : -INFINITY;
        s[t][2 + e] = (j >= low_b || sink) && j < high_b ? s[t][2 + e] * scale : -INFINITY;
        na = fmaxf(na, s[t][e]);
        nb = fmaxf(nb, s[t][2 + e]);
      }
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
      na = fmaxf(na, __shfl_xor_sync(0xffffffffu, na, x));
      nb = fmaxf(nb, __shfl_xor_sync(0xffffffffu, nb, x));
    }
    // The sums refer to the exact maxima: the largest weight, which has the most say, is then a
    // power of two and rounds to 16 bits without an error. Once the maxima have settled nothing is rescaled.
    const bool ga = na > ma, gb = nb > mb;
    if (__any_sync(0xffffffffu, ga || gb)) {
      const float fa = ga ? exp2_fast(ma - na) : 1.0f, fb = gb ? exp2_fast(mb - nb) : 1.0f;
      if (ga) ma = na;
      if (gb) mb = nb;
      la *= fa, lb *= fb;
#pragma unroll
      for (int i = 0; i < DP / 8; i++) o[i][0] *= fa, o[i][1] *= fa, o[i][2] *= fb, o[i][3] *= fb;
    }
    // a row that has seen nothing yet keeps a zero reference
    const float za = ma == -INFINITY ? 0.0f : ma - kRoom, zb = mb == -INFINITY ? 0.0f : mb - kRoom;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        s[t][e] = exp2_fast(s[t][e] - za);
        s[t][2 + e] = exp2_fast(s[t][2 + e] - zb);
        la += s[t][e], lb += s[t][2 + e];
      }
    const uint32_t pf[4] = {pack2<BF16>(s[0][0], s[0][1]), pack2<BF16>(s[0][2], s[0][3]),
                            pack2<BF16>(s[1][0], s[1][1]), pack2<BF16>(s[1][2], s[1][3])};
    // Where a key is hidden from one row and seen by another, 0 * v must stay 0 for the
    // first: values that are not finite are left out of the product and added for the rows
    // that see them.
    const int at_key = key_of(key);
    const bool mixed = __any_sync(0xffffffffu, low_a > at_key || high_a < at_key + kChunk ||
                                                   low_b > at_key || high_b < at_key + kChunk);
    bool wild = false;
    {
      const int r = (lane & 7) + (((lane >> 3) & 1) << 3);
#pragma unroll
      for (int n = 0; n < DP / 16; n++) {
        uint32_t b[4];
        const int v = 2 * n + (lane >> 4);
        ldm4t(vt + at(r, v), b);
        if (mixed)
#pragma unroll
          for (int i = 0; i < 4; i++) b[i] = zero_not_finite<BF16>(b[i], wild);
        mma16816<BF16>(o[2 * n], pf, b[0], b[1]);
        mma16816<BF16>(o[2 * n + 1], pf, b[2], b[3]);
      }
    }
    if (mixed && __any_sync(0xffffffffu, wild)) {
      for (int r = 0; r < kChunk; r++) {
        const bool sink = MODE == kChunks && at_key + r < sinks;
        const bool sees_a = (at_key + r >= low_a || sink) && at_key + r < high_a;
        const bool sees_b = (at_key + r >= low_b || sink) && at_key + r < high_b;
#pragma unroll
        for (int n = 0; n < DP / 8; n++) {
          uint32_t w;
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w)
                       : "r"(vt + at(r, n) + (lane & 3) * 4));
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const uint16_t x = (uint16_t)(w >> (16 * e));
            if (!not_finite<BF16>(x)) continue;
            if (sees_a) o[n][e] += to_float<BF16>(x);
            if (sees_b) o[n][2 + e] += to_float<BF16>(x);
          }
        }
      }
    }
    if (++stage == kStages) stage = 0, parity ^= 1;
  }
  if (MODE == kPrompt) asm volatile("cp.async.wait_group 0;");
  if (MODE != kPrompt && largest >= (uint32_t)c.pages && lane == 0) atomicOr(c.status, DM_KV_BAD_TOKEN);

  // ---- join the warps' states in shared memory
#pragma unroll
  for (int x = 1; x < 4; x <<= 1) {
    la += __shfl_xor_sync(0xffffffffu, la, x);
    lb += __shfl_xor_sync(0xffffffffu, lb, x);
  }
  __syncthreads();
  float *join = reinterpret_cast<float *>(smem) + warp * kRows * DP;
#pragma unroll
  for (int n = 0; n < DP / 8; n++) {
    const int col = n * 8 + (lane & 3) * 2;
    *reinterpret_cast<float2 *>(join + ra * DP + col) = make_float2(o[n][0], o[n][1]);
    *reinterpret_cast<float2 *>(join + rb8 * DP + col) = make_float2(o[n][2], o[n][3]);
  }
  if ((lane & 3) == 0) {
    sh.ml[warp][ra] = make_float2(ma - kRoom, la);
    sh.ml[warp][rb8] = make_float2(mb - kRoom, lb);
  }
  __syncthreads();
  // All of it is done before the kernel after this one may read the parts of both.
  if (beside) wait_for_previous();
  const bool final = MODE == kPrompt || d.part.parts == 1 || d.joins;
  constexpr int kLanes = DP / 4;  // threads along a row, four columns each
  const int col = (tid % kLanes) * 4;
  const float *all = reinterpret_cast<const float *>(smem);
  const int parts = MODE == kOwn && d.joins ? d.first_part : 0;  // of the shared keys
  for (int r = tid / kLanes; r < kRows; r += kThreads / kLanes) {
    if (sh.q[r] < 0) continue;
    // all loads first: there are few parts, and one after the other costs a microsecond each
    const float *part = d.part.o + sh.index[r] * dim + col;
    float2 ml[kMostJoined];
    float4 u[kMostJoined];
    if (MODE == kOwn) {
#pragma unroll
      for (int i = 0; i < kMostJoined; i++) {
        ml[i] = make_float2(-INFINITY, 0.0f);
        u[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (i < parts) {
          ml[i] = d.part.ml[i * d.part.rows + sh.index[r]];
          if (col < dim) u[i] = *reinterpret_cast<const float4 *>(part + i * d.part.rows * dim);
        }
      }
    }
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; w++) m = fmaxf(m, sh.ml[w][r].x);
    if (MODE == kOwn)
#pragma unroll
      for (int i = 0; i < kMostJoined; i++) m = fmaxf(m, ml[i].x);
    const float z = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWarps; w++)
      add_state(l, v, sh.ml[w][r], *reinterpret_cast<const float4 *>(all + (w * kRows + r) * DP + col), z);
    if (MODE == kOwn)
#pragma unroll
      for (int i = 0; i < kMostJoined; i++)
        if (ml[i].y != 0.0f) add_state(l, v, ml[i], u[i], z);  // else nothing was written
    if (final) {
      float *lse = kPacked ? p.lse : d.lse;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      if (col < dim) {
        uint16_t *out = (kPacked ? p.out : d.out) + sh.out[r] + col;
        *reinterpret_cast<uint2 *>(out) =
            make_uint2(pack2<BF16>(v.x * inv, v.y * inv), pack2<BF16>(v.z * inv, v.w * inv));
      }
      if (lse && col == 0) lse[sh.index[r]] = l == 0.0f ? -INFINITY : (m + log2_fast(l)) * kLn2;
    } else {
      const int64_t at = (int64_t)(d.first_part + blockIdx.y) * d.part.rows + sh.index[r];
      if (col < dim && l != 0.0f) *reinterpret_cast<float4 *>(d.part.o + at * dim + col) = v;
      if (col == 0) d.part.ml[at] = make_float2(m, l);
    }
  }
}

// ---------------------------------------------------------------------------
// Join the parts of each row: one block per row. Bound by the latency of two dependent loads
// and, with many parts, by their bytes.
// ---------------------------------------------------------------------------

// Chunks: a row that no entry owns has no parts.
template <bool BF16>
__global__ void __launch_bounds__(kJoinThreads)
join_kernel(const __grid_constant__ DecodeArgs d, const int32_t *offsets, int entries, int dim) {
  constexpr int kWarps = kJoinThreads / 32;
  __shared__ float top[kWarps], sum[kWarps], factor[kMostParts];
  __shared__ float4 acc[kWarps][64];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, parts = d.part.parts;
  wait_for_previous();
  let_next_start();
  if (offsets && (row / d.heads < offsets[0] || row / d.heads >= offsets[entries])) return;
  float2 ml[kMostParts / kJoinThreads];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kMostParts / kJoinThreads; k++) {
    const int i = tid + k * kJoinThreads;
    ml[k] = i < parts ? d.part.ml[i * d.part.rows + row] : make_float2(-INFINITY, 0.0f);
    m = fmaxf(m, ml[k].x);
  }
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
  if (lane == 0) top[warp] = m;
  __syncthreads();
  m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  const float z = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
#pragma unroll
  for (int k = 0; k < kMostParts / kJoinThreads; k++) {
    // a part that has seen nothing was not written
    const float f = ml[k].y == 0.0f ? 0.0f : exp2_fast(ml[k].x - z);
    l += ml[k].y * f;
    factor[tid + k * kJoinThreads] = f;
  }
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
  if (lane == 0) sum[warp] = l;
  __syncthreads();
  l = sum[0] + sum[1] + sum[2] + sum[3];
  float4 v[2] = {};
  const float *part = d.part.o + row * dim + lane * 4;
#pragma unroll 4
  for (int i = warp; i < parts; i += kWarps) {
    const float f = factor[i];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      float4 u = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (f != 0.0f && h * 128 + lane * 4 < dim)
        u = *reinterpret_cast<const float4 *>(part + i * d.part.rows * dim + h * 128);
      v[h].x += u.x * f, v[h].y += u.y * f, v[h].z += u.z * f, v[h].w += u.w * f;
    }
  }
  acc[warp][lane] = v[0];
  acc[warp][32 + lane] = v[1];
  __syncthreads();
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (tid < 64 && tid * 4 < dim) {
    float4 s = acc[0][tid];
    for (int w = 1; w < kWarps; w++) {
      const float4 u = acc[w][tid];
      s.x += u.x, s.y += u.y, s.z += u.z, s.w += u.w;
    }
    const int64_t b = row / d.heads, head = row % d.heads;
    uint16_t *out = d.out + b * d.out_stride[0] + head * d.out_stride[1] + tid * 4;
    *reinterpret_cast<uint2 *>(out) =
        make_uint2(pack2<BF16>(s.x * inv, s.y * inv), pack2<BF16>(s.z * inv, s.w * inv));
  }
  if (tid == 0 && d.lse) d.lse[row] = l == 0.0f ? -INFINITY : (m + log2_fast(l)) * kLn2;
}

// The same with a warp to a row, for many rows of few parts: bound by memory, where a block to a
// row is bound by the blocks (48000 rows of dim 128 in 2 parts 54 us longer than this one's 17).
constexpr int kFewParts = 8, kRowWarps = 8, kFewRows = 1024;

template <bool BF16>
__global__ void __launch_bounds__(kRowWarps * 32)
join_few_kernel(const __grid_constant__ DecodeArgs d, const int32_t *offsets, int entries, int dim) {
  const int64_t row = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, parts = d.part.parts;
  wait_for_previous();
  let_next_start();
  if (row >= d.part.rows || row / d.heads < offsets[0] || row / d.heads >= offsets[entries]) return;
  const float2 ml = lane < parts ? d.part.ml[lane * d.part.rows + row] : make_float2(-INFINITY, 0.0f);
  float m = ml.x;
#pragma unroll
  for (int x = 1; x < kFewParts; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
  m = __shfl_sync(0xffffffffu, m, 0);
  // a part that has seen nothing was not written
  const float mine = ml.y == 0.0f ? 0.0f : exp2_fast(ml.x - (m == -INFINITY ? 0.0f : m));
  float l = ml.y * mine;
#pragma unroll
  for (int x = 1; x < kFewParts; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
  l = __shfl_sync(0xffffffffu, l, 0);
  float4 v[2] = {};
  const float *part = d.part.o + row * dim + lane * 4;
#pragma unroll
  for (int i = 0; i < kFewParts; i++) {
    const float f = __shfl_sync(0xffffffffu, mine, i);
    if (i >= parts || f == 0.0f) continue;
#pragma unroll
    for (int h = 0; h < 2; h++)
      if (h * 128 + lane * 4 < dim) {
        const float4 u = *reinterpret_cast<const float4 *>(part + i * d.part.rows * dim + h * 128);
        v[h].x += u.x * f, v[h].y += u.y * f, v[h].z += u.z * f, v[h].w += u.w * f;
      }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t token = row / d.heads, head = row % d.heads;
  uint16_t *out = d.out + token * d.out_stride[0] + head * d.out_stride[1] + lane * 4;
#pragma unroll
  for (int h = 0; h < 2; h++)
    if (h * 128 + lane * 4 < dim)
      *reinterpret_cast<uint2 *>(out + h * 128) =
          make_uint2(pack2<BF16>(v[h].x * inv, v[h].y * inv), pack2<BF16>(v[h].z * inv, v[h].w * inv));
  if (lane == 0 && d.lse) d.lse[row] = l == 0.0f ? -INFINITY : (m + log2_fast(l)) * kLn2;
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

template <int MODE, int DP, int WARPS, bool BF16>
int32_t launch_rows(dim3 grid, const CUtensorMap *maps, const PromptArgs &p, const DecodeArgs &d,
                    const KvView &c, cudaStream_t s) {
  using Cfg = RowsCfg<DP, WARPS>;
  auto fn = rows_kernel<MODE, DP, WARPS, BF16>;
  DM_CUDA(dm::ensure_smem_limit((const void *)fn), "attention shared memory");
  return launch_chained("attention launch", fn, grid, Cfg::kThreads, Cfg::kSmem, s, maps[0], maps[1], p, d, c);
}

template <int MODE, int WARPS>
int32_t launch_rows(int type, int dim, dim3 grid, const CUtensorMap *maps, const PromptArgs &p,
                    const DecodeArgs &d, const KvView &c, cudaStream_t s) {
  const bool bf = type == DM_BF16;
  if (dim <= 64)
    return bf ? launch_rows<MODE, 64, WARPS, true>(grid, maps, p, d, c, s)
              : launch_rows<MODE, 64, WARPS, false>(grid, maps, p, d, c, s);
  if (dim <= 128)
    return bf ? launch_rows<MODE, 128, WARPS, true>(grid, maps, p, d, c, s)
              : launch_rows<MODE, 128, WARPS, false>(grid, maps, p, d, c, s);
  return bf ? launch_rows<MODE, 256, 4, true>(grid, maps, p, d, c, s)
            : launch_rows<MODE, 256, 4, false>(grid, maps, p, d, c, s);
}

// How a decode call is cut into parts. The workspace holds one state per part and row.
struct DecodePlan {
  bool tiles = false;  // the shared part runs on tcgen05 tiles
  bool wide = false;   // own keys: eight warps a block
  bool joins = false;  // the own part joins the shared ones
  int shared = 0;      // tokens that are read once for all; the rest is each sequence's own
  int shared_splits = 0, shared_parts = 0, own_parts = 0;
  int parts() const { return shared_parts + own_parts; }
};

constexpr int kSms = 148;
// The shared part runs on tiles where its rows fill more than one block of 16 and those blocks
// would read more than 12 MB of keys and values (each reads them all). 8 key/value heads of
// dim 128, us of 16-row blocks and of tiles: 24 to 192 rows a head on 256 tokens (2 to 13 MB)
// 12 to 21 and 14 to 27; 24 to 96 rows on 1216 (20 to 60 MB) 21 to 24 and 17 to 21; 128 rows
// on 9728 (319 MB) 61 and 41. One block of rows reads what tiles would: 16 rows on 32768
// tokens take 48 and 52.
constexpr int64_t kMostRowsBytes = 12 << 20;
constexpr int kSplitKeys = 128;  // a block's keys at least, where there are several
constexpr int kTileRows = 128;   // of a unit on tcgen05 tiles

// Blocks that cut `items` rows of blocks along `keys`: as many as run at once, no more (a
// second round costs more than shorter blocks save).
int splits_of(int64_t items, int keys, int64_t at_once) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(at_once / items, (keys + kSplitKeys - 1) / kSplitKeys));
}

// Microseconds on one B200, as measured: a block of tiles has 9 besides 1.2 for each step of
// its units beside blocks of rows (alone 0.95; dim above 128: 1.1 with pages of 64 tokens, 2.0
// with 16, taken as 1.6 for all); a block of rows 7 besides 0.9 (1.2) for each chunk of every
// warp, and beside tiles they get done 0.7 of what they would alone; a join in place 2; the join
// kernel 4 besides 0.4 for each MB of parts; a third launch 2.
constexpr float kTileUs = 9.0f, kTileStepUs = 1.2f, kTileStepWideUs = 1.6f, kRowsUs = 7.0f, kRowsStepUs = 0.9f,
                kRowsStepWideUs = 1.2f, kBeside = 0.7f, kInPlaceUs = 2.0f, kJoinUs = 4.0f, kJoinMbUs = 0.4f,
                kThirdUs = 2.0f;

DecodePlan decode_plan(int kv_heads, int heads, int dim, int batch, int shared, int max_length) {
  DecodePlan plan;
  if (batch == 0) return plan;
  const int group = heads / kv_heads;
  const bool has_own = max_length > shared || shared == 0;
  const int own = std::max(1, max_length - shared);
  const int64_t own_items = (int64_t)batch * kv_heads * ((group + kRows - 1) / kRows);
  // Blocks of eight warps have an SM to themselves, two of four warps share one: the first
  // are sooner done, where all of them run at once.
  plan.wide = dim <= 128 && own_items <= kSms;
  const int per_sm = plan.wide || dim > 128 ? 1 : 2, warps = plan.wide ? 8 : 4, at_once = kSms * per_sm;
  const float step = dim > 128 ? kRowsStepWideUs : kRowsStepUs;
  auto rows_us = [&](int keys, int warps) { return kRowsUs + step * ((keys + 16 * warps - 1) / (16 * warps)); };
  auto join_us = [&](int parts) { return kJoinUs + kJoinMbUs * parts * ((float)batch * heads * dim * 4e-6f); };

  // Each sequence reads all of its tokens: one launch, or two. With 32 and 8 heads of dim 128
  // and 64 shared tokens 13 us instead of 17 for 16 sequences, 21 instead of 24 for 64 (one
  // launch less; the caller's side 15.8 instead of 17.8), with 1056 for one 15 and 15 (20 and
  // 17.8); but 49 instead of 32 for 16 sequences with 4128.
  DecodePlan alone = plan;
  float alone_us = 0.0f;
  const int most_parts = splits_of(own_items, std::max(1, max_length), at_once);
  for (int parts : {1, most_parts}) {
    const float us = std::max(1.0f, (float)own_items / at_once) * rows_us((max_length + parts - 1) / parts, warps) +
                     (parts > 1 ? join_us(parts) : 0.0f);
    if (parts == 1 || us < alone_us) {
      alone_us = us;
      alone.own_parts = parts;
    }
  }
  if (shared == 0) return alone;

  // The shared tokens once for all, then what is left: two launches, or three.
  plan.shared = shared;
  if (has_own) plan.own_parts = splits_of(own_items, own, at_once);
  const int64_t row_blocks = ((int64_t)batch * group + kRows - 1) / kRows;
  plan.tiles = row_blocks > 1 && group <= 128 && kv_heads * row_blocks * shared * dim * 4 > kMostRowsBytes;
  float best = 0.0f;
  if (!plan.tiles) {
    const int64_t items = kv_heads * row_blocks;
    plan.shared_parts = plan.shared_splits = splits_of(items, shared, (dim > 128 ? 1 : 2) * kSms);
    plan.joins = plan.own_parts == 1 && plan.shared_parts <= kMostJoined;
    const float blocks = (float)items * plan.shared_splits;
    best = std::max(1.0f, blocks / ((dim > 128 ? 1 : 2) * kSms)) *
           rows_us((shared + plan.shared_splits - 1) / plan.shared_splits, 4);
    if (has_own) {
      const float one = rows_us((own + plan.own_parts - 1) / plan.own_parts, warps);
      // beside the shared blocks, if they leave room, else behind them
      const float left = plan.wide || dim > 128 ? kSms - blocks : at_once - blocks;
      best = (float)own_items * plan.own_parts <= left ? std::max(best, one)
                                                      : best + one * std::max(1.0f, (float)own_items / at_once);
    }
    best += plan.joins ? kInPlaceUs : plan.parts() > 1 ? join_us(plan.parts()) : 0.0f;
  } else {
    // More parts: shorter blocks, fewer SMs for the own part beside them, more to join.
    const int units = tile_shared_alternates(dim, group, batch) ? 2 : 1;
    const int tiles = (shared + tile_keys(dim) - 1) / tile_keys(dim);
    const int items = tile_shared_items(dim, kv_heads, group, batch);
    const int most = std::max(1, std::min(kSms / items, tiles / units));
    DecodePlan at = plan;
    for (int splits = 1, next = 1; splits <= most; splits += next, next = splits / 8 + 1) {
      at.shared_splits = splits;
      at.shared_parts = splits * units;
      const int per = (tiles + splits - 1) / splits;
      float us = kTileUs + (dim > 128 ? kTileStepWideUs : kTileStepUs) * ((per + units - 1) / units);
      const int left = kSms - std::min(kSms, items * splits);  // SMs beside the tiles
      if (has_own) {
        // own blocks are cut for the SMs that are left, if that leaves enough
        at.own_parts = splits_of(own_items, own, (int64_t)(left >= kSms / 2 ? left : kSms) * per_sm);
        const float blocks = (float)own_items * at.own_parts;
        const float one = rows_us((own + at.own_parts - 1) / at.own_parts, warps);
        at.joins = at.own_parts == 1 && at.shared_parts <= kMostJoined;
        if (blocks <= left * per_sm) {
          us = std::max(us, one);
        } else {  // what the tiles leave time for, then on all SMs; blocks that join wait for them
          float done = kBeside * left * per_sm * (us / one);
          if (at.joins) done = std::min(done, (float)left * per_sm);
          us += std::max(0.0f, blocks - done) / at_once * one;
          us = std::max(us, one);
        }
      }
      us += at.joins ? kInPlaceUs : at.parts() > 1 ? join_us(at.parts()) : 0.0f;
      if (splits == 1 || us < best) {
        best = us;
        plan = at;
      }
    }
  }
  if (has_own && !plan.joins) best += kThirdUs;
  return alone_us < best ? alone : plan;
}

uint64_t decode_workspace(const DecodePlan &plan, int64_t rows, int dim) {
  return plan.parts() > 1 ? (uint64_t)plan.parts() * rows * (dim * 4 + 8) : 0;
}

// How a call on chunks of new tokens is cut.
struct ChunkPlan {
  bool tiles = false;  // on tcgen05 tiles, else on blocks of 16 rows
  bool wide = false;   // these: eight warps a block
  int splits = 1;      // of each item's keys
};

// Microseconds on one B200, as measured, for a tile of one unit's rows (where memory does not set the
// rate, which it does whatever the cut) and of two (80 keys of dim 128, 128 of the others; dim 256
// with pages of 64 tokens and of 16), and for what an item of a block has besides. The rest is as in
// decode.
constexpr float kChunkStepUs[3][2] = {{0.8f, 1.6f}, {0.8f, 1.05f}, {1.6f, 2.05f}}, kChunkItemUs = 2.0f;
constexpr float kGain = 0.95f;  // more parts have to be worth their workspace
constexpr int64_t kMostPartBytes = 128 << 20;

// The host knows bounds only: entries, their rows together, the longest one's keys. Entries are
// taken to be alike.
ChunkPlan chunk_plan(const dm_kv_cache_desc &c, int heads, int entries, int64_t tokens, int max_length, int window,
                     int sinks) {
  ChunkPlan best;
  if (tokens == 0 || entries == 0) return best;
  const int dim = c.head_dim, group = heads / c.kv_heads;
  const int64_t busy = std::min<int64_t>(entries, tokens), each = (tokens + busy - 1) / busy;
  const int64_t part_bytes = tokens * heads * dim * 4;
  // what the rows of a block or unit see
  auto keys_of = [&](int64_t rows) {
    return (int)std::max<int64_t>(1, window ? std::min<int64_t>(max_length, (int64_t)window + sinks + rows) : max_length);
  };
  auto join_us = [&](int parts) { return parts > 1 ? kJoinUs + kJoinMbUs * 1e-6f * parts * part_bytes : 0.0f; };
  float best_us = 0.0f;
  auto offer = [&](const ChunkPlan &plan, float us) {
    if (plan.splits > 1 && plan.splits * part_bytes > kMostPartBytes) return;
    if (best_us == 0.0f || us < best_us * (plan.splits > best.splits ? kGain : 1.0f)) best = plan, best_us = us;
  };
  {
    const int64_t blocks = busy * ((each * group + kRows - 1) / kRows) * c.kv_heads;
    const int keys = keys_of(kRows / group);
    ChunkPlan plan;
    plan.wide = dim <= 128 && blocks <= kSms;
    const int at_once = kSms * (plan.wide || dim > 128 ? 1 : 2), warps = plan.wide ? 8 : 4;
    const float step = dim > 128 ? kRowsStepWideUs : kRowsStepUs;
    const int most = splits_of(blocks, keys, at_once);
    for (int splits : {1, most}) {
      plan.splits = splits;
      const int64_t rounds = (blocks * splits + at_once - 1) / at_once;
      offer(plan, rounds * (kRowsUs + step * ((keys + 16 * warps * splits - 1) / (16 * warps * splits))) + join_us(splits));
    }
  }
  const int64_t per = tile_chunk_tokens(dim, group);
  const int64_t items = busy * ((each + per - 1) / per) * c.kv_heads;
  const int tiles = (keys_of(std::min(each, per)) + tile_keys(dim) - 1) / tile_keys(dim);
  const bool second = dim > 128 ? c.page_tokens < 64 : each > kTileRows / group;
  const float step = kChunkStepUs[dim <= 64 ? 0 : dim <= 128 ? 1 : 2][second];
  ChunkPlan plan;
  plan.tiles = true;
  const int most = (int)std::max<int64_t>(1, std::min<int64_t>(std::max<int64_t>(2 * kSms / items, 4), std::min(tiles / 2, kMostParts)));
  for (plan.splits = 1; plan.splits <= most; plan.splits++) {
    const int64_t rounds = (items * plan.splits + kSms - 1) / kSms;
    offer(plan, kTileUs + rounds * step * ((tiles + plan.splits - 1) / plan.splits) + (rounds - 1) * kChunkItemUs +
                    join_us(plan.splits));
  }
  return best;
}

uint64_t chunk_workspace(const ChunkPlan &plan, int64_t rows, int dim) {
  return plan.splits > 1 ? (uint64_t)plan.splits * rows * (dim * 4 + 8) : 0;
}

}  // namespace dma

using namespace dma;

// A caller's bound on lengths, and what a row of the page table holds.
static int32_t bounded_length(const dm_kv_cache_desc &d, int32_t max_length) {
  return (int32_t)std::min<int64_t>(max_length, (int64_t)d.max_pages * d.page_tokens);
}

// Every tile of a prompt looks for its sequence among all, 32 at a time: half a microsecond for each.
constexpr int32_t kMostSequences = 1 << 20;

int32_t dma::check_strides(const int64_t *given, int64_t heads, int dim, int64_t *use, const char *what) {
  const bool none = given[0] == 0 && given[1] == 0;
  use[0] = none ? heads * dim : given[0];
  use[1] = none ? dim : given[1];
  if (use[0] % 8 || use[1] % 8)
    return fail(DM_ERR_INVALID_ARGUMENT, "%s strides must be multiples of 8 elements", what);
  if (use[0] < 0 || use[1] < 0) return fail(DM_ERR_INVALID_ARGUMENT, "%s strides are negative", what);
  return DM_OK;
}

int32_t dma::check_scale(float given, int dim, float *use) {
  if (!std::isfinite(given) || given < 0.0f)
    return fail(DM_ERR_POSITIVE_PARAMETER, "attention needs a finite scale that is not negative");
  *use = (given == 0.0f ? 1.0f / std::sqrt((float)dim) : given) * kLog2e;
  return DM_OK;
}

extern "C" {

int32_t dm_attention_prompt(dm_cuda_context *ctx, const dm_attention_prompt_desc *in, void *stream) {
  if (!ctx || !in) return fail(DM_ERR_INVALID_ARGUMENT, "null argument");
  if (in->type != DM_BF16 && in->type != DM_F16)
    return fail(DM_ERR_UNSUPPORTED_TENSOR_TYPE, "attention takes bf16 or f16");
  if (in->heads <= 0 || in->kv_heads <= 0 || in->heads % in->kv_heads || in->heads / in->kv_heads > 128)
    return fail(DM_ERR_ELEMENT_COUNT, "%d query heads over %d key/value heads", in->heads, in->kv_heads);
  if (in->kv_heads > 65535) return fail(DM_ERR_ELEMENT_COUNT, "%d key/value heads", in->kv_heads);
  if (in->head_dim <= 0 || in->head_dim % 8 || in->head_dim > 256)
    return fail(DM_ERR_ELEMENT_COUNT, "head_dim %d is not a multiple of 8 up to 256", in->head_dim);
  if (in->sequences < 0 || in->sequences > kMostSequences || in->window < 0)
    return fail(DM_ERR_ELEMENT_COUNT, "%d sequences, window %d", in->sequences, in->window);
  if (in->q_tokens < 0 || in->k_tokens < 0 || in->q_tokens > kMostTokens || in->k_tokens > kMostTokens)
    return fail(DM_ERR_ELEMENT_COUNT, "a bad number of tokens");
  if (in->sequences == 0 || in->q_tokens == 0) return DM_OK;
  if (!in->q || !in->out || !in->q_offsets || (in->k_tokens && (!in->k || !in->v)))
    return fail(DM_ERR_INVALID_ARGUMENT, "null tensor");
  if (((uintptr_t)in->q | (uintptr_t)in->k | (uintptr_t)in->v | (uintptr_t)in->out) & 15)
    return fail(DM_ERR_INVALID_ARGUMENT, "attention tensors must be 16-byte aligned");
  PromptArgs a{};
  a.q = (const uint16_t *)in->q;
  a.k = (const uint16_t *)in->k;
  a.v = (const uint16_t *)in->v;
  a.out = (uint16_t *)in->out;
  a.lse = in->lse;
  if (int32_t rc = check_strides(in->q_stride, in->heads, in->head_dim, a.q_stride, "query")) return rc;
  if (int32_t rc = check_strides(in->k_stride, in->kv_heads, in->head_dim, a.k_stride, "key")) return rc;
  if (int32_t rc = check_strides(in->v_stride, in->kv_heads, in->head_dim, a.v_stride, "value")) return rc;
  if (int32_t rc = check_strides(in->out_stride, in->heads, in->head_dim, a.out_stride, "output")) return rc;
  if (int32_t rc = check_scale(in->scale, in->head_dim, &a.scale)) return rc;
  a.q_offsets = in->q_offsets;
  a.k_offsets = in->k_offsets ? in->k_offsets : in->q_offsets;
  a.q_tokens = in->q_tokens;
  a.k_tokens = in->k_tokens;
  a.heads = in->heads;
  a.kv_heads = in->kv_heads;
  a.group = in->heads / in->kv_heads;
  a.dim = in->head_dim;
  a.sequences = in->sequences;
  a.causal = in->causal;
  a.window = in->window;
  cudaSetDevice(ctx->device);
  if (tile_prompt_fits(a)) return launch_tile_prompt(in->type, a, ctx, (cudaStream_t)stream);
  const int64_t tiles = in->q_tokens * a.group / kRows + in->sequences;
  if (tiles > INT32_MAX) return fail(DM_ERR_OVERFLOW, "too many query rows");
  const CUtensorMap none[2]{};
  return launch_rows<kPrompt, 4>(in->type, in->head_dim, dim3((unsigned)tiles, in->kv_heads), none, a,
                                 DecodeArgs{}, KvView{}, (cudaStream_t)stream);
}

int32_t dm_attention_decode_workspace(const dm_kv_cache *cache, int32_t heads, int32_t batch,
                                      int32_t shared_tokens, int32_t max_length, uint64_t *bytes) {
  if (!cache || !bytes) return fail(DM_ERR_INVALID_ARGUMENT, "null argument");
  const dm_kv_cache_desc &d = cache->desc;
  if (heads <= 0 || heads % d.kv_heads)
    return fail(DM_ERR_ELEMENT_COUNT, "%d query heads over %d key/value heads", heads, d.kv_heads);
  if (batch < 0 || (int64_t)batch * heads > (1 << 24))
    return fail(DM_ERR_ELEMENT_COUNT, "a batch of %d", batch);
  if (shared_tokens < 0 || shared_tokens % d.page_tokens || shared_tokens > (int64_t)d.max_pages * d.page_tokens)
    return fail(DM_ERR_ELEMENT_COUNT, "%d shared tokens are no whole pages of the table", shared_tokens);
  if (max_length < 0) return fail(DM_ERR_ELEMENT_COUNT, "max_length %d", max_length);
  *bytes = decode_workspace(decode_plan(d.kv_heads, heads, d.head_dim, batch, shared_tokens,
                                        bounded_length(d, max_length)),
                            (int64_t)batch * heads, d.head_dim);
  return DM_OK;
}

int32_t dm_attention_decode(dm_kv_cache *cache, const dm_attention_decode_desc *in, void *stream) {
  if (!cache || !in) return fail(DM_ERR_INVALID_ARGUMENT, "null argument");
  const dm_kv_cache_desc &kd = cache->desc;
  uint64_t need = 0;
  if (int32_t rc = dm_attention_decode_workspace(cache, in->heads, in->batch, in->shared_tokens,
                                                 in->max_length, &need))
    return rc;
  if (in->layer < 0 || in->layer >= kd.layers)
    return fail(DM_ERR_INVALID_LAYER, "layer %d of %d", in->layer, kd.layers);
  if (in->window < 0) return fail(DM_ERR_ELEMENT_COUNT, "window %d", in->window);
  if (in->batch == 0) return DM_OK;
  if (!in->q || !in->out) return fail(DM_ERR_INVALID_ARGUMENT, "null tensor");
  if (((uintptr_t)in->q | (uintptr_t)in->out) & 15)
    return fail(DM_ERR_INVALID_ARGUMENT, "attention tensors must be 16-byte aligned");
  if (need && (!in->workspace || ((uintptr_t)in->workspace & 15)))
    return fail(DM_ERR_INVALID_ARGUMENT, "decode needs a 16-byte aligned workspace");
  if (in->workspace_bytes < need)
    return fail(DM_ERR_BYTE_LENGTH, "a workspace of %llu bytes, %llu are needed",
                (unsigned long long)in->workspace_bytes, (unsigned long long)need);
  DecodeArgs a{};
  a.q = (const uint16_t *)in->q;
  a.out = (uint16_t *)in->out;
  a.lse = in->lse;
  if (int32_t rc = check_strides(in->q_stride, in->heads, kd.head_dim, a.q_stride, "query")) return rc;
  if (int32_t rc = check_strides(in->out_stride, in->heads, kd.head_dim, a.out_stride, "output")) return rc;
  if (int32_t rc = check_scale(in->scale, kd.head_dim, &a.scale)) return rc;
  a.sequences = in->sequences;
  a.heads = in->heads;
  a.group = in->heads / kd.kv_heads;
  a.batch = in->batch;
  a.layer = in->layer;
  a.window = in->window;
  a.max_length = bounded_length(kd, in->max_length);
  const DecodePlan plan = decode_plan(kd.kv_heads, in->heads, kd.head_dim, in->batch, in->shared_tokens, a.max_length);
  a.shared = plan.shared;
  a.part.parts = plan.parts();
  a.part.rows = (int64_t)in->batch * in->heads;
  a.part.o = (float *)in->workspace;
  a.part.ml = (float2 *)(a.part.o + (int64_t)a.part.parts * a.part.rows * kd.head_dim);
  cudaSetDevice(cache->ctx->device);
  cudaStream_t s = (cudaStream_t)stream;
  a.timeout = cache->ctx->status + kStatusWord;
  a.wait_limit = wait_limit(cache->ctx);
  CUtensorMap maps[2];
  if ((plan.own_parts || !plan.tiles) && !describe_chunks(kd.type, cache->view, in->layer, kChunk, maps))
    return fail(DM_ERR_COMMAND, "could not describe the cache for TMA");
  if (plan.shared_splits) {
    const int64_t items = (int64_t)kd.kv_heads * (((int64_t)in->batch * a.group + kRows - 1) / kRows);
    a.first_part = 0;
    a.splits = plan.shared_splits;
    if (int32_t rc = plan.tiles ? launch_tile_shared(kd.type, a, cache->view, s)
                                : launch_rows<kShared, 4>(kd.type, kd.head_dim, dim3((unsigned)items, a.splits), maps,
                                                      PromptArgs{}, a, cache->view, s))
      return rc;
  }
  if (plan.own_parts) {
    const int64_t items = (int64_t)in->batch * kd.kv_heads * ((a.group + kRows - 1) / kRows);
    a.first_part = plan.shared_parts;
    a.splits = plan.own_parts;
    a.joins = plan.joins;
    const dim3 grid((unsigned)items, a.splits);
    if (int32_t rc = plan.wide ? launch_rows<kOwn, 8>(kd.type, kd.head_dim, grid, maps, PromptArgs{}, a, cache->view, s)
                               : launch_rows<kOwn, 4>(kd.type, kd.head_dim, grid, maps, PromptArgs{}, a, cache->view, s))
      return rc;
  }
  if (plan.parts() > 1 && !a.joins)
    return launch_chained("attention join launch", kd.type == DM_BF16 ? join_kernel<true> : join_kernel<false>,
                          dim3((unsigned)a.part.rows), kJoinThreads, 0, s, a, (const int32_t *)nullptr, 0, kd.head_dim);
  return DM_OK;
}

// What both chunk calls look at.
static int32_t check_chunk(const dm_kv_cache *cache, const dm_attention_chunk_desc *in, dma::ChunkPlan *plan,
                           uint64_t *bytes) {
  if (!cache || !in) return fail(DM_ERR_INVALID_ARGUMENT, "null argument");
  const dm_kv_cache_desc &d = cache->desc;
  if (in->heads <= 0 || in->heads % d.kv_heads || in->heads / d.kv_heads > 128)
    return fail(DM_ERR_ELEMENT_COUNT, "%d query heads over %d key/value heads", in->heads, d.kv_heads);
  if (in->sequences < 0 || in->sequences > kMostSequences)
    return fail(DM_ERR_ELEMENT_COUNT, "%d sequences", in->sequences);
  if (in->window < 0 || in->sinks < 0)
    return fail(DM_ERR_ELEMENT_COUNT, "window %d, %d sinks", in->window, in->sinks);
  if (in->max_length < 0) return fail(DM_ERR_ELEMENT_COUNT, "max_length %d", in->max_length);
  if (in->tokens < 0 || in->tokens > kMostTokens) return fail(DM_ERR_ELEMENT_COUNT, "a bad number of tokens");
  const int64_t rows = in->tokens * in->heads;
  const int64_t tiles = chunk_tiles(in->tokens, in->sequences, in->heads / d.kv_heads, kRows);
  if (rows > INT32_MAX || tiles > INT32_MAX / d.kv_heads) return fail(DM_ERR_OVERFLOW, "too many query rows");
  *plan = chunk_plan(d, in->heads, in->sequences, in->tokens,
                     bounded_length(d, in->max_length), in->window, in->sinks);
  *bytes = chunk_workspace(*plan, rows, d.head_dim);
  return DM_OK;
}

int32_t dm_attention_chunk_workspace(const dm_kv_cache *cache, const dm_attention_chunk_desc *in, uint64_t *bytes) {
  if (!bytes) return fail(DM_ERR_INVALID_ARGUMENT, "null argument");
  ChunkPlan plan;
  return check_chunk(cache, in, &plan, bytes);
}

int32_t dm_attention_chunk(dm_kv_cache *cache, const dm_attention_chunk_desc *in, void *stream) {
  ChunkPlan plan;
  uint64_t need = 0;
  if (int32_t rc = check_chunk(cache, in, &plan, &need)) return rc;
  const dm_kv_cache_desc &kd = cache->desc;
  if (in->layer < 0 || in->layer >= kd.layers)
    return fail(DM_ERR_INVALID_LAYER, "layer %d of %d", in->layer, kd.layers);
  if (in->tokens == 0 || in->sequences == 0) return DM_OK;
  if (!in->q || !in->out || !in->offsets) return fail(DM_ERR_INVALID_ARGUMENT, "null tensor");
  if (((uintptr_t)in->q | (uintptr_t)in->out) & 15)
    return fail(DM_ERR_INVALID_ARGUMENT, "attention tensors must be 16-byte aligned");
  if (need && (!in->workspace || ((uintptr_t)in->workspace & 15)))
    return fail(DM_ERR_INVALID_ARGUMENT, "chunks need a 16-byte aligned workspace");
  if (in->workspace_bytes < need)
    return fail(DM_ERR_BYTE_LENGTH, "a workspace of %llu bytes, %llu are needed",
                (unsigned long long)in->workspace_bytes, (unsigned long long)need);
  PromptArgs p{};
  p.q = (const uint16_t *)in->q;
  p.out = (uint16_t *)in->out;
  p.lse = in->lse;
  if (int32_t rc = check_strides(in->q_stride, in->heads, kd.head_dim, p.q_stride, "query")) return rc;
  if (int32_t rc = check_strides(in->out_stride, in->heads, kd.head_dim, p.out_stride, "output")) return rc;
  if (int32_t rc = check_scale(in->scale, kd.head_dim, &p.scale)) return rc;
  p.q_offsets = p.k_offsets = in->offsets;
  p.q_tokens = p.k_tokens = in->tokens;
  p.heads = in->heads;
  p.kv_heads = kd.kv_heads;
  p.group = in->heads / kd.kv_heads;
  p.dim = kd.head_dim;
  p.sequences = in->sequences;
  p.causal = 1;
  p.window = in->window;
  p.sinks = in->sinks;
  DecodeArgs a{};
  a.out = p.out;
  a.lse = p.lse;
  a.out_stride[0] = p.out_stride[0];
  a.out_stride[1] = p.out_stride[1];
  a.sequences = in->rows;
  a.heads = in->heads;
  a.layer = in->layer;
  a.max_length = bounded_length(kd, in->max_length);
  a.splits = a.part.parts = plan.splits;
  a.part.rows = in->tokens * in->heads;
  a.part.o = (float *)in->workspace;
  a.part.ml = (float2 *)(a.part.o + (int64_t)a.part.parts * a.part.rows * kd.head_dim);
  a.timeout = cache->ctx->status + kStatusWord;
  a.wait_limit = wait_limit(cache->ctx);
  cudaSetDevice(cache->ctx->device);
  cudaStream_t s = (cudaStream_t)stream;
  CUtensorMap maps[2];
  const bool on_tiles = plan.tiles && tile_queries_fit(p.q_stride, p.group);
  if (!on_tiles && !describe_chunks(kd.type, cache->view, in->layer, kChunk, maps))
    return fail(DM_ERR_COMMAND, "could not describe the cache for TMA");
  const int64_t tiles = chunk_tiles(in->tokens, in->sequences, p.group, kRows);
  const dim3 grid((unsigned)(tiles * kd.kv_heads), plan.splits);
  if (int32_t rc = on_tiles  ? launch_tile_chunks(kd.type, p, a, cache->view, s)
                   : plan.wide ? launch_rows<kChunks, 8>(kd.type, kd.head_dim, grid, maps, p, a, cache->view, s)
                             : launch_rows<kChunks, 4>(kd.type, kd.head_dim, grid, maps, p, a, cache->view, s))
    return rc;
  if (plan.splits > 1 && plan.splits <= kFewParts && a.part.rows > kFewRows)
    return launch_chained("attention join launch", kd.type == DM_BF16 ? join_few_kernel<true> : join_few_kernel<false>,
                          dim3((unsigned)((a.part.rows + kRowWarps - 1) / kRowWarps)), kRowWarps * 32, 0, s, a,
                          in->offsets, in->sequences, kd.head_dim);
  if (plan.splits > 1)
    return launch_chained("attention join launch", kd.type == DM_BF16 ? join_kernel<true> : join_kernel<false>,
                          dim3((unsigned)a.part.rows), kJoinThreads, 0, s, a, in->offsets, in->sequences, kd.head_dim);
  return DM_OK;
}

}  // extern "C"
