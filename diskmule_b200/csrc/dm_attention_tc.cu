// dm_attention_tc.cu -- attention on tcgen05 tiles: 128 query rows against 128 keys.
//
// A block holds one or two units. A unit is 128 query rows (whole groups of query heads of
// one key/value head: row = token * group + head) with its own scores S [128 x 128 f32],
// weights P (16-bit, over S in tensor memory) and output sum O [128 x dim f32]. Per tile:
//   S = Q K^T       tcgen05.mma, both operands in shared memory (128-byte swizzle, TMA)
//   P = 2^(S - m)   one thread per row: maximum, exponentials, sum, all f32
//   O += P V        tcgen05.mma, P in tensor memory, V as it lies (keys down, dim across)
// m is the running maximum with slack: O and l are rescaled only where the maximum has grown
// by more than 2^8 since m was taken; until then the weights of newer keys may reach 2^8,
// which changes no relative rounding, and the common factor leaves in o / l.
//
// Up to dim 128 two units alternate on the tensor pipe: while one computes its exponentials
// the other's products run, and both read the same K and V tiles. For dim 256, O takes half
// of tensor memory, so one unit runs with two S buffers and the products of the next tile
// run under the exponentials of this one.
//
// Warps: 4 per unit softmax and output; then TMA, MMA issue, and two that keep values that
// are not finite out of tiles in which some key is hidden from some row (0 * NaN): they
// zero them in shared memory, and the output step adds them for the rows that see them.
#include <cudaTypedefs.h>

#include <algorithm>

#include "dm_attention.cuh"
#include "dm_attention_tc.cuh"
#include "dm_tcgen05.cuh"

using dmi::fail;

namespace dma {

using namespace dm::tc;

namespace {

constexpr int kUnitRows = 128, kTileKeys = 128;
constexpr int kStatusWord = 32;  // of the context's status buffer: a bounded wait ran out

template <int DP>
struct TcCfg {
  static constexpr int kUnits = DP == 256 ? 1 : 2;
  static constexpr int kBuffers = DP == 256 ? 2 : 1;         // S buffers of a unit
  static constexpr int kSoftWarps = 4 * kUnits;
  static constexpr int kThreads = (kSoftWarps + 4) * 32;
  static constexpr int kSlab = 128 * 128;                    // 128 rows x 64 values
  static constexpr int kTile = DP / 64 * kSlab;              // a Q, K or V tile
  static constexpr int kSlots = DP == 64 ? 8 : DP == 128 ? 4 : 2;  // ring of K and V tiles
  static constexpr int kSmem = 1024 + (kUnits + kSlots) * kTile;
  static constexpr int kOutCol = 256;                        // O in tensor memory; S before it
};

struct TcSmem {
  uint64_t q_full[2], s_full[2], p_full[2], pv_done[2];
  // K and V tiles: loaded; a V tile that is mixed has `dirty` in place of `full` for loaded,
  // and `clean` for fit to use; `empty` when its last product is done. K takes the even slots.
  uint64_t full[8], empty[8], dirty[8], clean[8], drain;
  uint32_t tmem;
  volatile int abort;
  int wild;      // a hidden-somewhere tile held values that are not finite
  int max_low, min_high, keys;
  TileOf tile;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int c0, int c1,
                                            int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3, %4, %5}], [%6];" ::"r"(dst),
      "l"((uint64_t)map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// 32 consecutive f32 columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float *r) {
  uint32_t *u = reinterpret_cast<uint32_t *>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]),
        "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]),
        "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]),
        "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]),
        "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(taddr));
}
// V [keys][64 values] slabs as the second operand with the values along N: 8-key groups lie
// 1024 bytes apart, 64-value slabs one slab apart.
__device__ __forceinline__ uint64_t v_desc(uint32_t addr, uint32_t slab) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(slab >> 4) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// 16-bit operands (bf16 or f16), f32 result, M = 128; N-major second operand for V
constexpr uint32_t idesc(bool bf16, int n, bool b_n_major) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_n_major ? 1u << 16 : 0u) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

enum TcMode { kTcPrompt, kTcShared };

struct TcArgs {
  PromptArgs p;
  DecodeArgs d;
  KvView c;
  int tokens;     // of a unit: 128 / group
  int tiles;      // prompt: upper bound of the number of tiles
  int alternate;  // shared: one unit's rows hold them all; the units take tiles in turn
  int32_t *timeout;
};

// What the roles of a block agree on.
struct Work {
  int kv_head, first, tiles;  // first key, number of key tiles
  int max_low, min_high, keys;
  int64_t k0;
  int table_row;
  __device__ bool mixed(int t) const {  // some row does not see some key of tile t
    const int key = first + t * kTileKeys;
    return key < max_low || key + kTileKeys > min_high;
  }
};

// One lane of a converged warp. What it decides is uniform, so the operands of the
// instructions under it can stay in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile(
      "{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(yes));
  return yes != 0;
}

// Bounded wait that also ends when another role has given up.
__device__ __forceinline__ bool wait(TcSmem &sh, uint64_t &bar, uint32_t parity) {
  const uint32_t b = smem_u32(&bar);
  if (mbar_try(b, parity)) return true;
  const long long start = clock64();
  while (!sh.abort) {
    if (mbar_try(b, parity)) return true;
    if (clock64() - start > kWaitCycles) break;
  }
  sh.abort = 1;
  return false;
}
// The same for a whole warp: one answer for all lanes.
__device__ __forceinline__ bool wait_warp(TcSmem &sh, uint64_t &bar, uint32_t parity) {
  return __all_sync(0xffffffffu, wait(sh, bar, parity));
}

// Two units: the 168 registers a thread that 384 threads start with, split anew (256 x 208 +
// 128 x 88 = 384 x 168), so that a row's 128 scores and the weights made from them stay in
// registers. Every warp of a group of four calls the same one.
__device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
}
__device__ __forceinline__ void give_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
}

template <int MODE, int DP, bool BF16>
__global__ void __launch_bounds__(TcCfg<DP>::kThreads, 1)
tile_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
            const __grid_constant__ CUtensorMap v_map, const __grid_constant__ TcArgs a) {
  using Cfg = TcCfg<DP>;
  constexpr int kUnits = Cfg::kUnits;
  extern __shared__ uint8_t raw[];
  __shared__ TcSmem sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
  const uint32_t ring = base + kUnits * Cfg::kTile;
  const int group = MODE == kTcPrompt ? a.p.group : a.d.group;
  const int per_unit = a.tokens * group;  // rows in use of a unit's 128

  // ---- which rows, which keys
  Work w{};
  int token0 = 0;  // first token (batch entry) of the block
  int lq = 0, lk = 0, split = 0;
  const int alternate = MODE == kTcShared && a.alternate;
  if (MODE == kTcPrompt) {
    // key/value heads side by side, the last (longest, if causal) tiles of the batch first
    w.kv_head = blockIdx.x % a.p.kv_heads;
    const int tile = a.tiles - 1 - blockIdx.x / a.p.kv_heads;
    if (warp == 0) {
      const TileOf t = find_tile(a.p.q_offsets, a.p.sequences, a.p.q_tokens, 1, kUnits * a.tokens, tile);
      if (lane == 0) sh.tile = t;
    }
  }
  if (tid == 0) {
    sh.abort = 0;
    sh.wild = 0;
    sh.max_low = 0, sh.min_high = INT32_MAX, sh.keys = 0;
    for (int i = 0; i < 2; i++) {
      mbar_init(smem_u32(&sh.q_full[i]), 1);
      mbar_init(smem_u32(&sh.s_full[i]), 1);
      mbar_init(smem_u32(&sh.p_full[i]), 4);
      mbar_init(smem_u32(&sh.pv_done[i]), 1);
    }
    for (int i = 0; i < Cfg::kSlots; i++) {
      mbar_init(smem_u32(&sh.full[i]), 1);
      mbar_init(smem_u32(&sh.empty[i]), 1);
      mbar_init(smem_u32(&sh.dirty[i]), 1);
      mbar_init(smem_u32(&sh.clean[i]), 2);
    }
    mbar_init(smem_u32(&sh.drain), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();

  // this thread's row, if it is a softmax thread
  const int unit = warp >> 2, row = tid & 127;
  const bool softmax = warp < Cfg::kSoftWarps;
  int low = 0, high = INT32_MAX;
  bool valid = false;
  int64_t out_at = 0, index = 0;
  if (MODE == kTcPrompt) {
    const TileOf t = sh.tile;
    if (t.seq < 0) return;
    w.k0 = min((int64_t)max(a.p.k_offsets[t.seq], 0), a.p.k_tokens);
    const int64_t k1 = min((int64_t)max(a.p.k_offsets[t.seq + 1], 0), a.p.k_tokens);
    lq = t.q1 - t.q0;
    lk = (int)max((int64_t)0, k1 - w.k0);
    token0 = t.tile * kUnits * a.tokens;
    const int last = min(lq, token0 + kUnits * a.tokens) - 1;
    // limits of the first and last token bound the others'
    auto low_of = [&](int i) { return a.p.window ? max(0, i + lk - lq - a.p.window + 1) : 0; };
    auto high_of = [&](int i) { return a.p.causal ? max(0, min(lk, i + lk - lq + 1)) : lk; };
    w.max_low = low_of(last);
    w.min_high = high_of(token0);
    w.keys = lk;
    w.first = low_of(token0) / kTileKeys * kTileKeys;
    const int end = high_of(last);
    w.tiles = end > w.first ? (end - w.first + kTileKeys - 1) / kTileKeys : 0;
    if (softmax) {
      const int token = token0 + unit * a.tokens + row / group;
      const int head = w.kv_head * group + row % group;
      valid = row < per_unit && token < lq;
      if (valid) {
        low = low_of(token), high = high_of(token);
        out_at = (t.q0 + (int64_t)token) * a.p.out_stride[0] + head * a.p.out_stride[1];
        index = (t.q0 + (int64_t)token) * a.p.heads + head;
      }
    }
    token0 += t.q0;
  } else {
    const int blocks = (a.d.batch + (alternate ? 1 : kUnits) * a.tokens - 1) / ((alternate ? 1 : kUnits) * a.tokens);
    const int rb = blockIdx.x % blocks;
    w.kv_head = blockIdx.x / blocks;
    split = blockIdx.y;
    token0 = rb * (alternate ? 1 : kUnits) * a.tokens;
    int unused;
    w.table_row = sequence_of(a.c, a.d, 0, &unused);
    if (softmax) {
      const int b = token0 + (alternate ? 0 : unit * a.tokens) + row / group;
      const int head = w.kv_head * group + row % group;
      valid = row < per_unit && b < a.d.batch;
      if (valid) {
        int length;
        sequence_of(a.c, a.d, b, &length);
        low = a.d.window ? max(0, length - a.d.window) : 0;
        high = min(length, a.d.shared);
        out_at = b * a.d.out_stride[0] + head * a.d.out_stride[1];
        index = (int64_t)b * a.d.heads + head;
      }
      const int top = __reduce_max_sync(0xffffffffu, valid ? low : 0);
      const int bottom = __reduce_min_sync(0xffffffffu, high);
      const int most = __reduce_max_sync(0xffffffffu, valid ? high : 0);
      if (lane == 0) {
        atomicMax(&sh.max_low, top);
        atomicMin(&sh.min_high, bottom);
        atomicMax(&sh.keys, most);
      }
    }
    __syncthreads();
    w.max_low = sh.max_low, w.min_high = sh.min_high, w.keys = sh.keys;
    const int all = (a.d.shared + kTileKeys - 1) / kTileKeys;
    const int per = (all + a.d.splits - 1) / a.d.splits;
    const int t0 = min(all, split * per), t1 = min((w.keys + kTileKeys - 1) / kTileKeys, t0 + per);
    w.first = t0 * kTileKeys;
    w.tiles = max(0, t1 - t0);
  }

  // tiles of unit u; its i-th is tile i, or 2 i + u when the units alternate
  auto count = [&](int u) -> int {
    if (alternate) return (w.tiles + 1 - u) / 2;
    if (MODE == kTcPrompt && kUnits == 2 && u == 0 && a.p.causal) {  // may need fewer
      const TileOf t = sh.tile;
      const int end = max(0, min(lk, min(lq, token0 - t.q0 + a.tokens) + lk - lq));
      return max(0, min(w.tiles, (end - w.first + kTileKeys - 1) / kTileKeys));
    }
    if (MODE == kTcPrompt && u == 1 && token0 - sh.tile.q0 + a.tokens >= lq) return 0;
    return w.tiles;
  };
  auto tile_of = [&](int u, int i) -> int { return alternate ? 2 * i + u : i; };
  const int n0 = count(0), n1 = kUnits == 2 ? count(1) : 0;

  if (warp == Cfg::kSoftWarps) tmem_alloc(smem_u32(&sh.tmem), 512);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;

  if (warp == Cfg::kSoftWarps) {
    // ---- TMA
    if (kUnits == 2) give_registers();
    if (w.tiles > 0) {
      if (lane == 0) {
        for (int u = 0; u < kUnits; u++) {
          if ((u ? n1 : n0) == 0) continue;
          const uint32_t bar = smem_u32(&sh.q_full[u]);
          mbar_expect_tx(bar, DP / 64 * per_unit * 128);
          for (int s = 0; s < DP / 64; s++)
            tma_load_4d(base + u * Cfg::kTile + s * Cfg::kSlab, &q_map, s * 64, 0, w.kv_head,
                        token0 + (alternate ? 0 : u * a.tokens), bar);
        }
      }
      int issued = 0;
      uint32_t parity = 0, dirty = 0;  // of the next load into a slot, by its barrier
      const int box = MODE == kTcShared ? min(a.c.page_tokens, kTileKeys) : kTileKeys;
      for (int i = 0; i < 2 * w.tiles; i++) {  // K and V of tile i / 2
        const int slot = i % Cfg::kSlots;
        const int key = w.first + (i >> 1) * kTileKeys;
        // pages of a tile: one lane each
        int page = 0, boxes = 1;
        if (MODE == kTcShared) {
          boxes = min(kTileKeys, a.d.shared - key) / box;
          if (lane < boxes) {
            const int p = a.c.table[(int64_t)w.table_row * a.c.max_pages + (key + lane * box) / a.c.page_tokens];
            page = (unsigned)p < (unsigned)a.c.pages ? p : a.c.pages;  // behind the map: zeros
          }
        }
        if (i >= Cfg::kSlots && !wait_warp(sh, sh.empty[slot], (i / Cfg::kSlots - 1) & 1)) break;
        const bool mixed = (i & 1) && w.mixed(i >> 1);
        const uint32_t bar = smem_u32(mixed ? &sh.dirty[slot] : &sh.full[slot]);
        (mixed ? dirty : parity) ^= 1u << slot;
        const CUtensorMap *map = i & 1 ? &v_map : &k_map;
        const uint32_t dst = ring + slot * Cfg::kTile;
        if (lane == 0) mbar_expect_tx(bar, DP / 64 * boxes * box * 128);
        __syncwarp();
        if (lane < boxes) {
          for (int s = 0; s < DP / 64; s++) {
            if (MODE == kTcPrompt)
              tma_load_3d(dst + s * Cfg::kSlab, map, s * 64, w.kv_head, (int)w.k0 + key, bar);
            else
              tma_load_4d(dst + s * Cfg::kSlab + lane * box * 128, map, s * 64,
                          (key + lane * box) % a.c.page_tokens, w.kv_head, page, bar);
          }
        }
        issued = i + 1;
      }
      if (sh.abort) {  // the copies in flight land before the block ends
        for (int i = max(0, issued - Cfg::kSlots); i < issued; i++) {
          const int slot = i % Cfg::kSlots;
          const bool mixed = (i & 1) && w.mixed(i >> 1);
          mbar_wait(smem_u32(mixed ? &sh.dirty[slot] : &sh.full[slot]),
                    (((mixed ? dirty : parity) >> slot) & 1) ^ 1);
        }
        for (int u = 0; u < kUnits; u++)
          if ((u ? n1 : n0) > 0) mbar_wait(smem_u32(&sh.q_full[u]), 0);
      }
    }
  } else if (warp == Cfg::kSoftWarps + 1) {
    // ---- MMA issue
    if (kUnits == 2) give_registers();
    // the whole warp follows the schedule, one lane issues
    if (w.tiles > 0) {
      constexpr uint32_t kQk = idesc(BF16, kTileKeys, false), kPv = idesc(BF16, DP, true);
      uint32_t full = 0, clean = 0;  // parity of the next V tile in a slot, by its barrier
      bool ok = true;
      const uint64_t q_desc = sw128_desc(base);
      auto products_s = [&](int u, int t, int buffer) {
        const uint64_t qd = q_desc + ((u * Cfg::kTile) >> 4);
        const uint64_t kd = sw128_desc(ring + ((2 * t) % Cfg::kSlots) * Cfg::kTile);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < DP / 16; k++) {
            const uint64_t at = (k / 4) * (Cfg::kSlab >> 4) + (k % 4) * 2;
            mma_ss(tmem + buffer * 128, qd + at, kd + at, kQk, k > 0);
          }
          mma_commit(smem_u32(&sh.s_full[buffer]));
        }
        __syncwarp();
      };
      auto products_o = [&](int u, int t, int buffer, bool add) {
        const uint64_t vd = v_desc(ring + ((2 * t + 1) % Cfg::kSlots) * Cfg::kTile, Cfg::kSlab);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < kTileKeys / 16; k++)
            mma_ts(tmem + Cfg::kOutCol + u * DP, tmem + buffer * 128 + k * 8, vd + k * (2048 >> 4), kPv,
                   add || k > 0);
          mma_commit(smem_u32(&sh.pv_done[u]));
        }
        __syncwarp();
      };
      auto k_there = [&](int t) {
        return wait_warp(sh, sh.full[(2 * t) % Cfg::kSlots], (2 * t / Cfg::kSlots) & 1);
      };
      // first of the units that use V tile t waits for it, in its clean form where mixed
      auto v_there = [&](int t, bool first_use) {
        if (!first_use) return true;
        const int slot = (2 * t + 1) % Cfg::kSlots;
        const bool mixed = w.mixed(t);
        uint32_t &parity = mixed ? clean : full;
        const uint32_t now = (parity >> slot) & 1;
        parity ^= 1u << slot;
        return wait_warp(sh, mixed ? sh.clean[slot] : sh.full[slot], now);
      };
      auto release = [&](int i) {
        if (elect_one()) mma_commit(smem_u32(&sh.empty[i % Cfg::kSlots]));
        __syncwarp();
      };
      if (kUnits == 2) {
        const int n[2] = {n0, n1};
        const int most = max(n0, n1);
#pragma unroll
        for (int u = 0; u < 2; u++) {
          if (n[u] == 0 || !ok) continue;
          const int t = tile_of(u, 0);
          ok = wait_warp(sh, sh.q_full[u], 0) && k_there(t);
          if (!ok) break;
          fence_after();
          products_s(u, t, u);
          if (alternate || u == 1 || n1 == 0) release(2 * t);
        }
        for (int i = 0; i < most && ok; i++) {
#pragma unroll
          for (int u = 0; u < 2; u++) {
            if (i >= n[u] || !ok) continue;
            const int t = tile_of(u, i);
            const bool first_use = alternate || u == 0 || i >= n0;
            ok = wait_warp(sh, sh.p_full[u], i & 1) && v_there(t, first_use);
            if (!ok) break;
            fence_after();
            products_o(u, t, u, i > 0);
            if (alternate || u == 1 || i >= n1) release(2 * t + 1);
            if (i + 1 < n[u]) {
              const int s = tile_of(u, i + 1);
              ok = k_there(s);
              if (!ok) break;
              fence_after();
              products_s(u, s, u);
              if (alternate || u == 1 || i + 1 >= n1) release(2 * s);
            }
          }
        }
      } else {
        ok = wait_warp(sh, sh.q_full[0], 0) && k_there(0);
        if (ok) {
          fence_after();
          products_s(0, 0, 0);
          release(0);
        }
        for (int t = 0; t < n0 && ok; t++) {
          if (t + 1 < n0) {
            ok = k_there(t + 1);
            if (!ok) break;
            fence_after();
            products_s(0, t + 1, (t + 1) & 1);
            release(2 * t + 2);
          }
          ok = wait_warp(sh, sh.p_full[t & 1], (t >> 1) & 1) && v_there(t, true);
          if (!ok) break;
          fence_after();
          products_o(0, t, t & 1, t > 0);
          release(2 * t + 1);
        }
      }
      if (!ok) {  // products in flight end before tensor memory is given back
        if (elect_one()) mma_commit(smem_u32(&sh.drain));
        mbar_wait(smem_u32(&sh.drain), 0);
      }
    }
    __syncwarp();
  } else if (warp >= Cfg::kSoftWarps + 2) {
    // ---- values that are not finite leave mixed tiles
    if (kUnits == 2) give_registers();
    const int who = tid - (Cfg::kSoftWarps + 2) * 32;
    uint32_t dirty = 0;  // parity of the next mixed tile in a slot
    for (int t = 0; t < w.tiles; t++) {
      if (!w.mixed(t)) continue;
      const int slot = (2 * t + 1) % Cfg::kSlots;
      const uint32_t parity = (dirty >> slot) & 1;
      dirty ^= 1u << slot;
      if (!wait_warp(sh, sh.dirty[slot], parity)) break;
      const uint32_t v = ring + slot * Cfg::kTile;
      constexpr uint32_t kExp = BF16 ? 0x7f807f80u : 0x7c007c00u;
      bool found = false;
#pragma unroll 4
      for (int i = who; i < Cfg::kTile / 16; i += 64) {
        const uint4 x = lds16(v + i * 16);
        const uint32_t hit = __vcmpeq2(x.x & kExp, kExp) | __vcmpeq2(x.y & kExp, kExp) |
                             __vcmpeq2(x.z & kExp, kExp) | __vcmpeq2(x.w & kExp, kExp);
        if (hit) {
          found = true;
          const uint32_t e[4] = {x.x & ~__vcmpeq2(x.x & kExp, kExp), x.y & ~__vcmpeq2(x.y & kExp, kExp),
                                 x.z & ~__vcmpeq2(x.z & kExp, kExp), x.w & ~__vcmpeq2(x.w & kExp, kExp)};
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(v + i * 16), "r"(e[0]),
                       "r"(e[1]), "r"(e[2]), "r"(e[3])
                       : "memory");
        }
      }
      if (found) sh.wild = 1;
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.clean[slot]));
    }
  } else {
    // ---- softmax: one thread per row
    if (kUnits == 2) take_registers();
    const int n = unit ? n1 : n0;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // TMEM lane of the warp's first row
    const uint32_t o_at = tmem + lanes + Cfg::kOutCol + unit * DP;
    const float c = MODE == kTcPrompt ? a.p.scale : a.d.scale;
    float m = -INFINITY, l = 0.0f;  // m in units of the raw score
    bool ok = true;
    for (int i = 0; i < n; i++) {
      const int buffer = kUnits == 2 ? unit : i & 1;
      const int phase = kUnits == 2 ? i : i >> 1;
      if (!(ok = wait_warp(sh, sh.s_full[buffer], phase & 1))) break;
      fence_after();
      const uint32_t s_at = tmem + lanes + buffer * 128;
      const int key = w.first + tile_of(unit, i) * kTileKeys;
      float x[128];
#pragma unroll
      for (int j = 0; j < 4; j++) tmem_ld32(s_at + 32 * j, x + 32 * j);
      tmem_wait_ld();
      const int from = low - key, to = high - key;  // columns [from, to) are visible
      if (__any_sync(0xffffffffu, from > 0 || to < kTileKeys)) {
#pragma unroll
        for (int j = 0; j < 128; j++) x[j] = j >= from && j < to ? x[j] : -INFINITY;
      }
      float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
      for (int j = 4; j < 128; j += 8)
#pragma unroll
        for (int k = 0; k < 4; k++)
          top[k] = j + 4 + k < 128 ? fmaxf(fmaxf(top[k], x[j + k]), x[j + 4 + k]) : fmaxf(top[k], x[j + k]);
      const float now = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
      // 2^8: the slack of the running maximum. Each row goes by its own scores alone.
      const bool grows = (now - m) * c > 8.0f;
      if (__any_sync(0xffffffffu, grows)) {
        const float f = grows ? exp2_fast((m - now) * c) : 1.0f;
        if (i > 0) {
          if (!(ok = wait_warp(sh, sh.pv_done[unit], (i - 1) & 1))) break;
          fence_after();
#pragma unroll 1
          for (int j = 0; j < DP; j += 16) {
            uint32_t o[16];
            tmem_ld16(o_at + j, o);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
            tmem_st16(o_at + j, o);
          }
        }
        l *= f;
        if (grows) m = now;
      }
      const float z = m == -INFINITY ? 0.0f : -m * c;
      const uint64_t cc = pair(c, c), zz = pair(z, z);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        uint32_t p[16];
#pragma unroll
        for (int k = 0; k < 16; k++) {
          const uint64_t e = fma2(pair(x[32 * j + 2 * k], x[32 * j + 2 * k + 1]), cc, zz);
          const float e0 = exp2_fast(__uint_as_float((uint32_t)e));
          const float e1 = exp2_fast(__uint_as_float((uint32_t)(e >> 32)));
          sum[k & 1] = add2(sum[k & 1], pair(e0, e1));
          p[k] = pack2<BF16>(e0, e1);
        }
        tmem_st16(s_at + 16 * j, p);
      }
      sum[0] = add2(sum[0], sum[1]);
      l += __uint_as_float((uint32_t)sum[0]) + __uint_as_float((uint32_t)(sum[0] >> 32));
      tmem_wait_st();
      // With two S buffers the product of step i - 1 may still run. Its barrier must not get
      // two phases ahead of this warp, so it is waited for before step i's can start.
      if (Cfg::kBuffers == 2 && i > 0 && !(ok = wait_warp(sh, sh.pv_done[unit], (i - 1) & 1))) break;
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[buffer]));
    }
    // ---- result
    if (ok && n > 0) ok = wait_warp(sh, sh.pv_done[unit], (n - 1) & 1);
    if (ok) {
      fence_after();
      const bool wild = n > 0 && sh.wild;
      const bool final = MODE == kTcPrompt || a.d.part.parts == 1;
      const int dim = MODE == kTcPrompt ? a.p.dim : a.c.head_dim;
      const float inv = !final ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
      const int64_t part_at =
          MODE == kTcShared
              ? (int64_t)(a.d.first_part + (alternate ? 2 * split + unit : split)) * a.d.part.rows + index
              : 0;
#pragma unroll 1
      for (int j = 0; j < DP; j += 32) {
        float o[32];
        __syncwarp();
        if (n > 0) {
          tmem_ld32(o_at + j, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int k = 0; k < 32; k++) o[k] = 0.0f;
        }
        if (wild && valid) {  // rare: what was left out of the products
          for (int i = 0; i < n; i++) {
            const int t = tile_of(unit, i), key = w.first + t * kTileKeys;
            if (!w.mixed(t)) continue;
            for (int r = max(key, low); r < min(key + kTileKeys, high); r++) {
              const uint16_t *v;
              if (MODE == kTcPrompt) {
                v = a.p.v + (w.k0 + r) * a.p.v_stride[0] + w.kv_head * a.p.v_stride[1];
              } else {
                const int page = a.c.table[(int64_t)w.table_row * a.c.max_pages + r / a.c.page_tokens];
                if ((unsigned)page >= (unsigned)a.c.pages) continue;
                v = reinterpret_cast<const uint16_t *>(
                        a.c.memory + page * a.c.page_bytes + a.d.layer * a.c.layer_bytes +
                        (a.c.kv_heads + w.kv_head) * a.c.head_bytes) +
                    (int64_t)(r % a.c.page_tokens) * dim;
              }
#pragma unroll
              for (int k = 0; k < 32; k++)
                if (j + k < dim && not_finite<BF16>(v[j + k])) o[k] += to_float<BF16>(v[j + k]);
            }
          }
        }
        if (valid && final) {
          uint16_t *out = (MODE == kTcPrompt ? a.p.out : a.d.out) + out_at + j;
#pragma unroll
          for (int k = 0; k < 32; k += 8)
            if (j + k < dim)
              *reinterpret_cast<uint4 *>(out + k) =
                  make_uint4(pack2<BF16>(o[k] * inv, o[k + 1] * inv), pack2<BF16>(o[k + 2] * inv, o[k + 3] * inv),
                             pack2<BF16>(o[k + 4] * inv, o[k + 5] * inv), pack2<BF16>(o[k + 6] * inv, o[k + 7] * inv));
        } else if (valid && l != 0.0f) {
          float *out = a.d.part.o + part_at * dim + j;
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            if (j + k < dim) *reinterpret_cast<float4 *>(out + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
        }
      }
      if (valid && final) {
        float *lse = MODE == kTcPrompt ? a.p.lse : a.d.lse;
        if (lse) lse[index] = l == 0.0f ? -INFINITY : (m * c + log2_fast(l)) * kLn2;
      } else if (valid) {
        a.d.part.ml[part_at] = make_float2(m * c, l);
      }
    }
  }
  fence_before();
  __syncthreads();
  if (tid == 0 && sh.abort) atomicExch(a.timeout, 1);
  if (warp == Cfg::kSoftWarps) {
    fence_after();
    tmem_dealloc(tmem, 512);
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void *p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (PFN_cuTensorMapEncodeTiled_v12000)p;
  }();
  return fn;
}

// A tensor map of 16-bit values with 64-value rows, 128-byte swizzle. Strides are in bytes,
// of dimension 1 and up; a dimension of one has none that matters.
bool encode(CUtensorMap *map, bool bf16, const void *base, int rank, const uint64_t *dims,
            const int64_t *strides, const uint32_t *box) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t d[4], s[3];
  cuuint32_t b[4], e[4] = {1, 1, 1, 1};
  for (int i = 0; i < rank; i++) {
    d[i] = dims[i];
    b[i] = box[i];
    if (i) s[i - 1] = dims[i] == 1 ? 16 : (cuuint64_t)strides[i - 1];
  }
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
            const_cast<void *>(base), d, s, b, e, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// q as {dim, head of a group, key/value head, token}; a box is one unit's rows
bool encode_q(CUtensorMap *map, bool bf16, const void *q, const int64_t *stride, int dim, int group,
              int kv_heads, int64_t tokens, int box_tokens) {
  const uint64_t dims[4] = {(uint64_t)dim, (uint64_t)group, (uint64_t)kv_heads, (uint64_t)tokens};
  const int64_t strides[3] = {stride[1] * 2, stride[1] * 2 * group, stride[0] * 2};
  const uint32_t box[4] = {64, (uint32_t)group, 1, (uint32_t)box_tokens};
  return encode(map, bf16, q, 4, dims, strides, box);
}

template <int MODE, int DP, bool BF16>
int32_t launch(dim3 grid, const CUtensorMap *maps, const TcArgs &a, cudaStream_t s) {
  auto fn = tile_kernel<MODE, DP, BF16>;
  static bool set = false;  // per instantiation; setting it twice is harmless
  if (!set) {
    DM_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, TcCfg<DP>::kSmem),
            "attention shared memory");
    set = true;
  }
  fn<<<grid, TcCfg<DP>::kThreads, TcCfg<DP>::kSmem, s>>>(maps[0], maps[1], maps[2], a);
  DM_CUDA(cudaGetLastError(), "attention launch");
  return DM_OK;
}

template <int MODE>
int32_t launch(bool bf16, int dim, dim3 grid, const CUtensorMap *maps, const TcArgs &a, cudaStream_t s) {
  if (dim <= 64)
    return bf16 ? launch<MODE, 64, true>(grid, maps, a, s) : launch<MODE, 64, false>(grid, maps, a, s);
  if (dim <= 128)
    return bf16 ? launch<MODE, 128, true>(grid, maps, a, s) : launch<MODE, 128, false>(grid, maps, a, s);
  return bf16 ? launch<MODE, 256, true>(grid, maps, a, s) : launch<MODE, 256, false>(grid, maps, a, s);
}

int units_of(int dim) { return dim > 128 ? 1 : 2; }

}  // namespace

bool tile_prompt_fits(const PromptArgs &p) {
  // a broadcast tensor (stride 0) has no tensor map
  for (const int64_t *s : {p.q_stride, p.k_stride, p.v_stride})
    if (s[0] <= 0 || s[1] <= 0 || s[0] >= (int64_t)1 << 37 || s[1] * p.group >= (int64_t)1 << 37) return false;
  return p.k_tokens > 0;
}

int32_t launch_tile_prompt(int32_t type, const PromptArgs &p, int32_t *status, cudaStream_t stream) {
  TcArgs a{};
  a.p = p;
  a.tokens = kUnitRows / p.group;
  a.timeout = status + kStatusWord;
  const int64_t tiles = p.q_tokens / (units_of(p.dim) * a.tokens) + p.sequences;
  if (tiles * p.kv_heads > INT32_MAX) return fail(DM_ERR_OVERFLOW, "too many query rows");
  a.tiles = (int)tiles;
  const bool bf16 = type == DM_BF16;
  CUtensorMap maps[3];
  const uint64_t dims[3] = {(uint64_t)p.dim, (uint64_t)p.kv_heads, (uint64_t)p.k_tokens};
  const uint32_t box[3] = {64, 1, (uint32_t)kTileKeys};
  const int64_t ks[2] = {p.k_stride[1] * 2, p.k_stride[0] * 2}, vs[2] = {p.v_stride[1] * 2, p.v_stride[0] * 2};
  if (!encode_q(&maps[0], bf16, p.q, p.q_stride, p.dim, p.group, p.kv_heads, p.q_tokens, a.tokens) ||
      !encode(&maps[1], bf16, p.k, 3, dims, ks, box) || !encode(&maps[2], bf16, p.v, 3, dims, vs, box))
    return fail(DM_ERR_COMMAND, "could not describe the attention tensors for TMA");
  return launch<kTcPrompt>(bf16, p.dim, dim3((unsigned)(tiles * p.kv_heads)), maps, a, stream);
}

bool tile_shared_alternates(int dim, int group, int batch) {
  return units_of(dim) == 2 && batch <= kUnitRows / group;
}

int tile_shared_items(int dim, int kv_heads, int group, int batch) {
  const int units = tile_shared_alternates(dim, group, batch) ? 1 : units_of(dim);
  const int per = units * (kUnitRows / group);
  return kv_heads * ((batch + per - 1) / per);
}

int32_t launch_tile_shared(int32_t type, const DecodeArgs &d, const KvView &c, int32_t *status,
                           cudaStream_t stream) {
  TcArgs a{};
  a.d = d;
  a.c = c;
  a.tokens = kUnitRows / d.group;
  a.alternate = tile_shared_alternates(c.head_dim, d.group, d.batch);
  a.timeout = status + kStatusWord;
  const bool bf16 = type == DM_BF16;
  CUtensorMap maps[3];
  const uint64_t dims[4] = {(uint64_t)c.head_dim, (uint64_t)c.page_tokens, (uint64_t)c.kv_heads, (uint64_t)c.pages};
  const int64_t strides[3] = {c.head_dim * 2, c.head_bytes, c.page_bytes};
  const uint32_t box[4] = {64, (uint32_t)std::min(c.page_tokens, kTileKeys), 1, 1};
  const uint8_t *k = c.memory + d.layer * c.layer_bytes, *v = k + c.kv_heads * c.head_bytes;
  if (!encode_q(&maps[0], bf16, d.q, d.q_stride, c.head_dim, d.group, c.kv_heads, d.batch, a.tokens) ||
      !encode(&maps[1], bf16, k, 4, dims, strides, box) || !encode(&maps[2], bf16, v, 4, dims, strides, box))
    return fail(DM_ERR_COMMAND, "could not describe the cache for TMA");
  const int items = tile_shared_items(c.head_dim, c.kv_heads, d.group, d.batch);
  return launch<kTcShared>(bf16, c.head_dim, dim3((unsigned)items, (unsigned)d.splits), maps, a, stream);
}

}  // namespace dma

extern "C" int32_t dm_attention_status(dm_cuda_context *ctx, void *stream) {
  if (!ctx) return fail(DM_ERR_INVALID_ARGUMENT, "null context");
  cudaSetDevice(ctx->device);
  int32_t bit = 0;
  cudaStream_t s = (cudaStream_t)stream;
  DM_CUDA(cudaMemcpyAsync(&bit, ctx->status + dma::kStatusWord, 4, cudaMemcpyDeviceToHost, s), "attention status");
  DM_CUDA(cudaMemsetAsync(ctx->status + dma::kStatusWord, 0, 4, s), "attention status");
  DM_CUDA(cudaStreamSynchronize(s), "attention status");
  if (bit) return fail(DM_ERR_TIMEOUT, "a bounded wait ran out in an attention kernel");
  return DM_OK;
}
