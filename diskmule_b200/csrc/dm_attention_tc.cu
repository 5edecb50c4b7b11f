// dm_attention_tc.cu -- attention on tcgen05 tiles: 128 query rows against a tile of keys.
//
// A block holds one or two units. A unit is 128 query rows (whole groups of query heads of
// one key/value head: row = token * group + head) with its own scores S [128 x keys f32],
// weights P (16-bit) and output sum O [128 x dim f32], all in tensor memory. Per tile:
//   S = Q K^T       tcgen05.mma, both operands in shared memory (128-byte swizzle, TMA)
//   P = 2^(S - m)   one thread per row (chunks of dim 256: two): maximum, exponentials, sum, all f32
//   O += P V        tcgen05.mma, P in tensor memory, V as it lies (keys down, dim across)
// m is the running maximum with slack: O and l are rescaled only where the maximum has grown
// by more than 2^8 since m was taken; until then the weights of newer keys may reach 2^8 (f16:
// 2^15, see kTileHeadroom), and the common factor leaves in o / l.
//
// The threads of a unit should never wait for products. So S of the next tile is computed
// while the weights of this one are: P has columns of its own beside S, and tensor memory
// (512 columns) sets the tile's keys. dim 64: 2 units of S 128 + P 64 + O 64. dim 128: 2 of
// S 80 + P 40 + O 128. dim 256: one of S 128 + two P of 64 + O 256 (the threads of a single
// unit are not to wait for its product either; with P in the place of two S in turn 8192 x
// 9472 tokens took 10% longer). Both units read the same K and V tiles.
//
// A block works through several items (prompt: 256 or 128 query rows; it takes over blocks
// that have not started yet), so that loads, first products and output of different items
// overlap. Every wait and every product costs its warp 100 cycles or more, so each job has
// warps of its own with a short loop: 4 per unit for softmax and output, one each for the
// products S and O of a unit, for the loads of K and of V, for the choice of items, and one
// that keeps values that are not finite out of tiles in which some key is hidden from some
// row (0 * NaN): it zeroes them in shared memory, and the output step adds them for the rows
// that see them. (At dim 128 one warp for all products of both units took 3600 cycles for 128
// keys, one per unit 4100; so it is 1750 for 80, 2800 for 128.)
//
// Weights are rounded to 16 bits, once, because both operands of a product have one type; the
// sum l takes them unrounded. They lie where the type has all its bits (f16: down to 2^-21 of the
// reference's), so each is off by half a unit in its last place: an error of the result that is
// no larger than its own rounding where one key has most of the weight, and averages out where
// many have.
//
// Chunks of new tokens over the cache (kTcChunks) are prompts whose keys lie in pages: boxes of whole
// pages or parts of them, looked up a tile ahead. Keys that no row of an item sees, between the sinks
// and its window, are left out of the numbering of its keys. Where there are few items their keys are
// cut in parts, which a kernel of its own joins. An item of one unit's rows at most (a single token, a
// draft, the end of a prompt) goes through both units, which take its tiles in turn, since one unit
// alone waits for each of its steps. Each unit then joins half of the dims from both sums, which it
// can read, as a row has the same lane of tensor memory in both (16 tokens over 20000, not cut: dim
// 128 231 us on one unit, 197 on two; dim 64 195 and 131).
// 4096 tokens over 28672, 16 heads of dim 128: 846 us by themselves, 1.22 PFLOP/s (two rounds of 256
// equal items on 148 SMs), 950 at the power limit; 2001 tokens over 6000 beside 30 single ones over
// 190 to 7643: 269 and 316 (295 and 334 with single tokens on one unit); 1500 tokens, window 1024 and
// 4 sinks, dim 256, with others 38. That is one round of items of 11 tiles, whose 62,500 cycles (1.67
// GHz) are 4300 until the item is found, 5000 until its first scores are there, 43,700 for the tiles
// (3800 for one that hides nothing and rescales nothing, 2150 of the threads and 1650 waiting for
// scores; 3300 to 4600 with hidden keys or rows whose maximum grows, which wait for the product before),
// 5000 for the last product and 4600 for the output; 5000 more from cold caches. Pages of 16, 64 or 256
// tokens make no difference; without sinks it is 33 us.
//
// Measured, causal 16384 tokens, 16 heads of dim 128: 807 us, 1.36 PFLOP/s; without a mask 8192
// keys, dim 256 1.47, dim 64 0.74. What bounds it: at dim 128, 1750 cycles a tile of both units,
// where the tensor pipe needs 1280 (1460 counting what S reads from shared memory: 6.5 KB for 40
// cycles of 16 values) and the exponential unit as many (each busy 60% of a run over 6144 tokens,
// the issue slots 41%), and power in long runs; at dim 64 the exponentials, 2048 of 2600 cycles
// for 128 keys; in short prompts 5000 cycles an item for the last product, the output's stores
// and the first tile.
#include <cudaTypedefs.h>

#include <algorithm>

#include "../../include/diskmule_selftest.h"
#include "dm_attention.cuh"
#include "dm_attention_tc.cuh"
#include "dm_tcgen05.cuh"

using dmi::fail;

namespace dma {

using namespace dm::tc;

namespace {

constexpr int kUnitRows = 128;
constexpr int kItems = 4;        // items between the first role and the last
constexpr int kMostSlots = 5;
constexpr int kJoinTiles = 2;    // of an item for two units to take in turn (64 items of two: 35 us, now 33)
constexpr int kWantTiles = 6;    // tiles left to load when the next item is chosen; at least 1

// SIDES: threads of a row, each with its part of a tile's keys and of the dims.
template <int DP, int SIDES = 1>
struct TcCfg {
  static constexpr int kUnits = DP == 256 ? 1 : 2;
  static constexpr int kKeys = DP == 128 ? 80 : 128;         // of a tile
  // warps
  static constexpr int kSoftWarps = 4 * kUnits * SIDES;
  static constexpr int kItemWarp = kSoftWarps, kKWarp = kItemWarp + 1, kVWarp = kItemWarp + 2;
  static constexpr int kScrubWarp = kItemWarp + 3;
  static constexpr int kSWarp = kItemWarp + 4;               // products S, one warp per unit
  static constexpr int kOWarp = kSWarp + kUnits;             // products O
  static constexpr int kThreads = kSoftWarps == 4 ? 384 : 512;  // whole groups of four warps
  // the warps behind the last one scrub too
  static constexpr int kScrubWarps = 1 + kThreads / 32 - (kOWarp + kUnits);
  static constexpr int kConsumers = kThreads / 32 - 1;       // of an item
  // K and V move in chunks, each in a ring of its own: whole tiles, or for dim 256 quarters
  // (64 values of all keys of K, 32 keys of V), so that a chunk's place is free again soon.
  static constexpr int kChunks = DP == 256 ? 4 : 1;          // of a tile
  static constexpr int kChunkBytes = kKeys * DP * 2 / kChunks;
  static constexpr int kVKeys = kKeys / kChunks;             // keys of a V chunk
  static constexpr int kKSlabs = DP / 64 / kChunks;          // 64-value slabs of a K chunk
  static constexpr int kSlots = DP == 128 ? 4 : 5;           // of a ring
  static constexpr int kQBytes = kUnitRows * DP * 2;
  static constexpr int kSmem = 1024 + kUnits * kQBytes + 2 * kSlots * kChunkBytes;  // beside TcSmem
  // columns of tensor memory
  static constexpr int kUnitCols = DP == 64 ? 192 : 128;     // S from unit to unit
  static constexpr int kPCol = kKeys;                        // P from S
  static constexpr int kOCol = DP == 64 ? 384 : 256;
  // Registers: the launch's share (128 or 168 a thread) split anew, so that a row's scores and
  // the weights made from them stay in registers: 256 x 192 + 256 x 64 = 512 x 128, and
  // 128 x 216 + 256 x 144 = 384 x 168. Two threads to a row have half the scores each: 256 x 160 +
  // 256 x 96 (192 and 64 spill in the other roles, and take 5% longer).
  static constexpr int kScaled = DP == 64 ? 32 : 64;         // columns of O rescaled at once
  static constexpr int kSoftRegs = kSoftWarps == 4 ? 216 : SIDES == 2 ? 160 : 192;
  static constexpr int kOtherRegs = kSoftWarps == 4 ? 144 : SIDES == 2 ? 96 : 64;
};

// What the roles know of an item.
struct Item {
  int stop, kv_head, first, tiles;  // first key, number of key tiles
  int n[2];                         // tiles of each unit
  int alternate;                    // one unit's rows are all there are: both have them, and take tiles in turn
  int max_low, min_high;            // every row sees the keys [max_low, min_high)
  int token0, lq, lk, q0, k0;       // first token of the item and of its sequence
  int table_row, end;               // paged: where its pages are looked up; no row sees keys from `end` on
  int split, sinks, gap;            // chunks: its part of the keys; numbers from `sinks` on are keys `gap` further
  int wild;                         // values that are not finite were found
};

struct TcSmem {
  uint64_t item_full[kItems], item_empty[kItems], next_block;
  uint64_t want;  // the item's last tiles are being loaded: time for the next item
  uint64_t q_full, q_empty, s_full[2], s_free[2];  // S by unit
  uint64_t p_full[2], pv_done[2];                  // weights: by unit, or the two of one unit
  // chunks: loaded; fit to use (V, by the scrub warp); all products done
  uint64_t k_full[kMostSlots], k_empty[kMostSlots];
  uint64_t v_full[kMostSlots], v_clean[kMostSlots], v_empty[kMostSlots], drain[4];
  uint64_t told[4], heard[4];  // both sides of a quarter of the rows have left word, and read the other's
  float word[2][kUnitRows];
  uint4 answer;  // which block was taken over
  Item item[kItems];
  uint32_t tmem;
  volatile int abort;
  volatile uint32_t loaded, asked, looked;  // signs of life: chunks of K, and blocks, asked for; entries looked at
};

static_assert(TcCfg<256>::kSmem + sizeof(TcSmem) <= 227 * 1024 && TcCfg<128>::kSmem + sizeof(TcSmem) <= 227 * 1024,
              "a block's shared memory");

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Ask for a block of this grid that has not started; the answer lands in shared memory.
__device__ __forceinline__ void take_block(uint32_t answer, uint32_t bar) {
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
          answer),
      "r"(bar)
      : "memory");
}
// The taken block's x index, or -1 when none was left.
__device__ __forceinline__ int taken_block(uint32_t answer) {
  uint32_t yes, x, y, z, w;
  asm volatile(
      "{\n .reg .b128 h;\n .reg .pred p;\n"
      " ld.shared.b128 h, [%5];\n"
      " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n"
      " selp.u32 %0, 1, 0, p;\n mov.u32 %1, 0;\n mov.u32 %2, 0;\n mov.u32 %3, 0;\n mov.u32 %4, 0;\n"
      " @p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, %2, %3, %4}, h;\n}\n"
      : "=r"(yes), "=r"(x), "=r"(y), "=r"(z), "=r"(w)
      : "r"(answer)
      : "memory");
  return yes ? (int)x : -1;
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
// 8 columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
      : "memory");
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

enum TcMode { kTcPrompt, kTcShared, kTcChunks };

struct TcArgs {
  PromptArgs p;
  DecodeArgs d;
  KvView c;
  int tokens;     // of a unit: 128 / group
  int tiles;      // prompt, chunks: upper bound of the number of items per key/value head
  int alternate;  // shared: one unit's rows hold them all; the units take tiles in turn
  int k_box, v_box;  // paged: rows of a TMA box
  int wide;          // rows of the result (or of the parts) lie on 32-byte boundaries
  int32_t *timeout;
  int64_t wait_limit;
};

// Bounded wait that also ends when another role has given up; one answer for the warp. A
// warp that waits sleeps in try_wait: one that polls takes issue slots from the softmax warps
// beside it (measured: a third of the prompt rate).
__device__ __forceinline__ bool wait(TcSmem &sh, int64_t limit, uint64_t &bar, uint32_t parity) {
  constexpr unsigned kAll = 0xffffffffu;
  const uint32_t b = smem_u32(&bar);
  if (__all_sync(kAll, mbar_look(b, parity))) return true;
  const long long start = clock64();
  bool done = false, stop = false;
  while (!done && !stop) {
    done = __all_sync(kAll, mbar_look(b, parity));
    stop = __any_sync(kAll, sh.abort || clock64() - start > limit);
  }
  if (!done) sh.abort = 1;
  return done;
}
// The same for what comes once in an item: the limit holds for a tile, and an item has any
// number of them, and so have the blocks without an item before it. So this goes on as long as
// the item's keys come in, or blocks or entries are gone through.
__device__ __forceinline__ bool wait_item(TcSmem &sh, int64_t limit, uint64_t &bar, uint32_t parity) {
  constexpr unsigned kAll = 0xffffffffu;
  const uint32_t b = smem_u32(&bar);
  long long start = clock64();
  uint32_t loaded = kAll;
  while (!__all_sync(kAll, mbar_look(b, parity))) {
    if (!__any_sync(kAll, sh.abort || clock64() - start > limit)) continue;
    const uint32_t now = __shfl_sync(kAll, sh.loaded + sh.asked + sh.looked, 0);
    if (__any_sync(kAll, sh.abort) || now == loaded) {
      sh.abort = 1;
      return false;
    }
    loaded = now;
    start = clock64();
  }
  return true;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// First key of tile t of an item; chunks number the keys without the gap behind the sinks.
template <int MODE, int KEYS>
__device__ __forceinline__ int key_of(const Item &w, int t) {
  const int number = w.first + t * KEYS;
  return MODE == kTcChunks && number >= w.sinks ? number + w.gap : number;
}
// Whether some row does not see some key of tile t.
template <int MODE, int KEYS>
__device__ __forceinline__ bool mixed(const Item &w, int t) {
  const int key = key_of<MODE, KEYS>(w, t);
  return key < w.max_low || key + KEYS > w.min_high;
}

template <int REGS>
__device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
}
template <int REGS>
__device__ __forceinline__ void give_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}

// A place in a ring: slot and how often the ring has been gone round.
template <int SLOTS>
struct Place {
  int slot = 0;
  uint32_t round = 0;
  __device__ void next() {
    if (++slot == SLOTS) slot = 0, round++;
  }
  __device__ uint32_t parity() const { return round & 1; }
  // the same slot, one round earlier
  __device__ void back(int n) {
    for (; n > 0; n--)
      if (--slot < 0) slot = SLOTS - 1, round--;
  }
};

// Where a block's search for items stands: at 32 entries in a step of the lengths, with `before` items
// before them. A block's items mostly ascend, so it looks at every entry four times in all (0.7 us for
// 32 of them), not for every item: 1024 entries of 8 tokens, 32 and 8 heads of dim 128, 2007 us, now
// 784; of 40 tokens, 16 and 2 heads of dim 256, 1698 and 993. Runs of entries without rows are passed
// over by a search (3 entries of up to 300 rows among 4096: 475 us with a look at each for every item,
// 375 at each four times, now 24).
struct ChunkSearch {
  int turn = 3, s0 = 0;
  int64_t before = 0;
};

// The last of offsets[low .. high], which ascend, that is at most q; offsets[low] is. One warp.
__device__ __forceinline__ int last_upto(const int32_t *offsets, int low, int high, int q) {
  const int lane = threadIdx.x & 31;
  for (int count = high - low + 1; count > 1;) {
    const int step = (count + 31) / 32, end = low + count;
    const int64_t at = low + (int64_t)lane * step;
    low += (__popc(__ballot_sync(0xffffffffu, at < end && offsets[at] <= q)) - 1) * step;
    count = min(step, end - low);
  }
  return low;
}

// Chunks: the items of `tokens` tokens in order of their sequences' lengths, in four steps of the
// longest, so that no long item begins when the others are done, and from a sequence's last on.
// One warp; as find_tile.
__device__ __forceinline__ TileOf find_chunk(const PromptArgs &p, const DecodeArgs &d, const KvView &c, int tokens,
                                             int64_t tile, ChunkSearch &at, volatile uint32_t &looked) {
  const int lane = threadIdx.x & 31;
  TileOf r{-1, 0, 0, 0, 0, 0, 0};
  const int step = d.max_length / 4 + 1;
  if (tile < at.before) at = ChunkSearch{};
  for (; at.turn >= 0; at.turn--, at.s0 = 0)
    for (; at.s0 < p.sequences; at.s0 += 32) {
      const int s = at.s0 + lane;
      int q0 = 0, q1 = 0, length = 0;
      if (s < p.sequences) {
        sequence_of(c, d, s, &length);
        q0 = p.q_offsets[s], q1 = p.q_offsets[s + 1];
        q0 = (int)min((int64_t)max(q0, 0), p.q_tokens), q1 = max(q0, (int)min((int64_t)q1, p.q_tokens));
      }
      if (lane == 0) looked = looked + 1;
      if (!__any_sync(0xffffffffu, q1 > q0)) {  // on with the next entry that has rows, if there is one
        const int q = __shfl_sync(0xffffffffu, q0, 0);
        at.s0 = (q < p.q_tokens ? last_upto(p.q_offsets, at.s0, p.sequences, q) : p.sequences) - 32;
        continue;
      }
      if (length / step != at.turn) q1 = q0;
      const int64_t n = ((int64_t)(q1 - q0) + tokens - 1) / tokens;
      int64_t upto = at.before + n;
      if (lane > 0) upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, tile < upto);
      if (hit) {
        const int src = __ffs(hit) - 1;
        r.seq = at.s0 + src;
        r.tile = (int)__shfl_sync(0xffffffffu, upto - 1 - tile, src);
        r.q0 = __shfl_sync(0xffffffffu, q0, src);
        r.q1 = __shfl_sync(0xffffffffu, q1, src);
        return r;
      }
      at.before = __shfl_sync(0xffffffffu, upto, 31);
    }
  r.behind = tile - at.before;
  return r;
}

// Load the K or V tiles of an item into the ring, chunk by chunk.
template <int MODE, int DP, bool V>
__device__ __forceinline__ bool load_tiles(TcSmem &sh, const Item &w, int tiles, const TcArgs &a,
                                           const CUtensorMap *map, uint32_t ring, uint32_t lead,
                                           Place<TcCfg<DP>::kSlots> &place) {
  using Cfg = TcCfg<DP>;
  constexpr int kRows = V ? Cfg::kVKeys : Cfg::kKeys;     // keys of a chunk
  constexpr int kSlabs = V ? DP / 64 : Cfg::kKSlabs;      // its slabs of 64 values
  const int lane = threadIdx.x & 31;
  const int kv_head = w.kv_head, k0 = w.k0, table_row = w.table_row, end = w.end;
  constexpr bool kPaged = MODE != kTcPrompt;
  // paged: a box lies in one page; lane i looks the tile's i-th up, a tile ahead. Boxes and
  // pages are powers of two or whole chunks.
  const int box = !kPaged ? kRows : V ? a.v_box : a.k_box;
  const int box_bits = 31 - __clz(box), most = kPaged ? kRows >> box_bits : 1, page_bits = 31 - __clz(a.c.page_tokens);
  auto looks = [&](int at) -> bool { return lane * box < Cfg::kKeys && at + lane * box < end; };
  // As the table has it: a number outside the pool is outside the map, too, and reads as zeros.
  // It is looked at a tile later, so that nothing waits for it, and reported at the end.
  uint32_t largest = 0;
  auto page_at = [&](int at) -> int {
    return looks(at) ? a.c.table[(int64_t)table_row * a.c.max_pages + ((at + lane * box) >> page_bits)] : -1;
  };
  // shared: all of the shared pages are there; else up to the last key
  const int most_keys = MODE == kTcShared ? a.d.shared : end;
  const int number0 = w.first, sinks = MODE == kTcChunks ? w.sinks : 0, gap = MODE == kTcChunks ? w.gap : 0;
  auto key_at = [&](int t) -> int {
    const int number = number0 + t * Cfg::kKeys;
    return MODE == kTcChunks && number >= sinks ? number + gap : number;
  };
  // the chunk's boxes, each in kSlabs slabs; one lane for each
  const int slab = lane % kSlabs, mine = lane / kSlabs;
  const uint32_t place_in = slab * kRows * 128 + mine * box * 128;
  int next_pages = kPaged && tiles > 0 ? page_at(key_at(0)) : 0;
  for (int t = 0; t < tiles; t++) {
    const int pages = next_pages, key = key_at(t);
    if (kPaged && !V && looks(key)) largest = max(largest, (uint32_t)pages);
    if (kPaged && t + 1 < tiles) next_pages = page_at(key_at(t + 1));
    // No sooner than it is needed: blocks that have not started are for whoever is done first.
    if (!V && t == max(0, tiles - kWantTiles) && lead) mbar_arrive(smem_u32(&sh.want));
    if (!V && lead) sh.loaded = place.round * TcCfg<DP>::kSlots + place.slot;
    // the same for all chunks of a tile of K
    int boxes = !kPaged ? 1 : min(most, max(0, most_keys - key + box - 1) >> box_bits);
    int page = kPaged ? __shfl_sync(0xffffffffu, pages, mine) : 0, row = (key + mine * box) & (a.c.page_tokens - 1);
#pragma unroll 1
    for (int c = 0; c < Cfg::kChunks; c++, place.next()) {
      const int x0 = V ? 0 : c * kSlabs * 64;
      if (V && kPaged && c > 0) {
        const int from = key + c * kRows;
        boxes = min(most, max(0, most_keys - from + box - 1) >> box_bits);
        page = __shfl_sync(0xffffffffu, pages, c * most + mine);
        row = (from + mine * box) & (a.c.page_tokens - 1);
      }
      const uint32_t bar = smem_u32(V ? &sh.v_full[place.slot] : &sh.k_full[place.slot]);
      const uint32_t dst = ring + place.slot * Cfg::kChunkBytes;
      uint64_t &empty = V ? sh.v_empty[place.slot] : sh.k_empty[place.slot];
      if (place.round > 0 && !wait(sh, a.wait_limit, empty, place.parity() ^ 1)) return false;
      if (lead) mbar_expect_tx(bar, kSlabs * boxes * box * 128);
      __syncwarp();
      if (MODE == kTcPrompt) {
        if (lane < kSlabs)
          tma_load_3d(dst + slab * kRows * 128, map, x0 + slab * 64, kv_head, k0 + key + (V ? c * kRows : 0), bar);
      } else if (mine < boxes) {
        tma_load_4d(dst + place_in, map, x0 + slab * 64, row, kv_head, page, bar);
      }
      __syncwarp();
    }
  }
  if (kPaged && !V && largest >= (uint32_t)a.c.pages) atomicOr(a.c.status, DM_KV_BAD_TOKEN);
  return true;
}

// A row's sides. One unit has four softmax warps, one a scheduler, and nothing beside them while they
// wait. Pages and sinks leave chunks of dim 256 with tiles of 3200 cycles then, where the products
// need 2050; with two threads to a row 2800 (1500 tokens, windows 1024 and 4096: 40 and 89 us, now 36
// and 77). A prompt's tile takes 2450 with one.
template <int MODE, int DP>
constexpr int kSidesOf = MODE == kTcChunks && DP == 256 ? 2 : 1;

template <int MODE, int DP, bool BF16>
__global__ void __launch_bounds__((TcCfg<DP, kSidesOf<MODE, DP>>::kThreads), 1)
tile_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
            const __grid_constant__ CUtensorMap v_map, const __grid_constant__ TcArgs a) {
  constexpr int kSides = kSidesOf<MODE, DP>;
  constexpr bool kJoins = MODE == kTcChunks && DP <= 128;  // units join what they have of one item
  using Cfg = TcCfg<DP, kSides>;
  constexpr int kUnits = Cfg::kUnits, kKeys = Cfg::kKeys, kChunks = Cfg::kChunks, kSlots = Cfg::kSlots;
  using Ring = Place<kSlots>;
  extern __shared__ uint8_t raw[];
  __shared__ TcSmem sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
  const uint32_t k_ring = base + kUnits * Cfg::kQBytes, v_ring = k_ring + kSlots * Cfg::kChunkBytes;
  constexpr bool kPacked = MODE != kTcShared;  // query rows by offsets
  const int group = kPacked ? a.p.group : a.d.group;
  const int per_unit = a.tokens * group;  // rows in use of a unit's 128
  const int split = MODE == kTcShared ? blockIdx.y : 0;
  // P of a unit's product `number`: which, and how often it has been used before
  auto p_of = [&](int u, int number) -> int { return kUnits == 2 ? u : number & 1; };
  auto p_round = [&](int number) -> int { return kUnits == 2 ? number : number >> 1; };
  auto tile_of = [&](int alternate, int u, int i) -> int { return alternate ? 2 * i + u : i; };
  // whether tile t of an item is one of the n of unit u
  auto is_mine = [&](int alternate, int u, int t, int n) -> bool { return alternate ? (t & 1) == u : t < n; };

  if (tid == 0) {
    sh.abort = 0;
    sh.loaded = sh.asked = sh.looked = 0;
    for (int i = 0; i < kItems; i++) {
      mbar_init(smem_u32(&sh.item_full[i]), 1);
      mbar_init(smem_u32(&sh.item_empty[i]), Cfg::kConsumers);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(smem_u32(&sh.s_full[i]), 1);
      mbar_init(smem_u32(&sh.s_free[i]), 4 * kSides);
      mbar_init(smem_u32(&sh.p_full[i]), 4 * kSides);
      mbar_init(smem_u32(&sh.pv_done[i]), 1);
    }
    for (int i = 0; i < kSlots; i++) {
      mbar_init(smem_u32(&sh.k_full[i]), 1);
      mbar_init(smem_u32(&sh.k_empty[i]), kUnits);
      mbar_init(smem_u32(&sh.v_full[i]), 1);
      mbar_init(smem_u32(&sh.v_clean[i]), Cfg::kScrubWarps);
      mbar_init(smem_u32(&sh.v_empty[i]), kUnits);
    }
    mbar_init(smem_u32(&sh.q_full), 1);
    mbar_init(smem_u32(&sh.q_empty), kUnits);
    mbar_init(smem_u32(&sh.next_block), 1);
    mbar_init(smem_u32(&sh.want), 1);
    for (int i = 0; i < 4; i++) {
      mbar_init(smem_u32(&sh.drain[i]), 1);
      mbar_init(smem_u32(&sh.told[i]), 2);
      mbar_init(smem_u32(&sh.heard[i]), 2);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == Cfg::kItemWarp) tmem_alloc(smem_u32(&sh.tmem), 512);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  // What a kernel after this one may read without waiting is older than this one's inputs.
  wait_for_previous();
  let_next_start();
  bool ok = true;  // of the role: no wait has run out

  if (warp >= Cfg::kSoftWarps) {
    give_registers<Cfg::kOtherRegs>();
    if (warp == Cfg::kItemWarp) {
      // ---- choice of items
      int block = blockIdx.x, items = 0, asks = 0;
      int64_t all = INT64_MAX;  // tiles of the batch, once a block has been behind them
      ChunkSearch search;
      while (ok) {
      Item w{};
      if (kPacked) {
        if (block < 0) {
          w.stop = 1;
        } else {
          // key/value heads side by side, the last (longest, if causal) tiles of the batch first,
          // chunks the longest sequences
          w.kv_head = block % a.p.kv_heads;
          const int splits = MODE == kTcChunks ? a.d.splits : 1, rest = block / a.p.kv_heads;
          w.split = rest % splits;
          const int tile = MODE == kTcChunks ? rest / splits : a.tiles - 1 - rest;
          TileOf t{-1};
          if (tile < all) {
            t = MODE == kTcChunks ? find_chunk(a.p, a.d, a.c, kUnits * a.tokens, tile, search, sh.looked)
                                  : find_tile(a.p, 1, kUnits * a.tokens, tile);
            if (t.seq < 0) all = tile - t.behind;
          }
          if (t.seq < 0) {
            w.stop = -1;  // behind the last tile
          } else {
            w.q0 = t.q0;
            w.k0 = t.k0;
            if (MODE == kTcChunks) w.table_row = sequence_of(a.c, a.d, t.seq, &w.lk);
            else w.lk = t.k1 - t.k0;
            const int lq = w.lq = t.q1 - t.q0, lk = w.lk;
            w.token0 = t.tile * kUnits * a.tokens;
            const int last = min(lq, w.token0 + kUnits * a.tokens) - 1;
            // limits of the first and last token bound the others'
            w.max_low = low_of(a.p, lq, lk, last);
            w.min_high = high_of(a.p, lq, lk, w.token0);
            const int low = low_of(a.p, lq, lk, w.token0), end = high_of(a.p, lq, lk, last);
            const int end0 = high_of(a.p, lq, lk, min(last, w.token0 + a.tokens - 1));  // of the first unit
            if (MODE == kTcChunks) {
              const Range r = range_of(a.p, low, end, kKeys);
              const int all = (r.keys + kKeys - 1) / kKeys, per = (all + splits - 1) / splits;
              const int t0 = min(all, w.split * per);
              w.end = end;
              w.sinks = r.sinks;
              w.gap = r.low - r.sinks;
              w.first = t0 * kKeys;
              w.tiles = min(all, t0 + per) - t0;
              const int upto = min(end0, r.sinks) + max(0, end0 - r.low);  // numbers below end0
              w.n[0] = min(w.tiles, max(0, (upto + kKeys - 1) / kKeys - t0));
            } else {
              w.first = low / 16 * 16;
              auto tiles_to = [&](int end) { return max(0, (end - w.first + kKeys - 1) / kKeys); };
              w.tiles = tiles_to(end);
              w.n[0] = tiles_to(end0);
            }
            w.n[1] = kUnits == 2 && w.token0 + a.tokens < lq ? w.tiles : 0;
            if (kJoins && w.n[1] == 0 && w.tiles >= kJoinTiles) {
              w.alternate = 1;
              w.n[0] = (w.tiles + 1) / 2;
              w.n[1] = w.tiles / 2;
            }
          }
        }
      } else if (items > 0) {
        w.stop = 1;
      } else {
        const int alternate = w.alternate = a.alternate, units = alternate ? 1 : kUnits;
        const int blocks = (a.d.batch + units * a.tokens - 1) / (units * a.tokens);
        w.kv_head = block / blocks;
        w.token0 = block % blocks * units * a.tokens;
        // Pages are looked up for the sequence that has most of the shared tokens: the others,
        // which may be shorter or empty, have the same pages as far as they reach and no
        // entries behind that.
        int top = 0, bottom = INT32_MAX, mine = 0, table_row = 0;
        for (int b = w.token0 + lane; b < min(a.d.batch, w.token0 + units * a.tokens); b += 32) {
          int length;
          const int row = sequence_of(a.c, a.d, b, &length), sees = min(length, a.d.shared);
          top = max(top, a.d.window ? max(0, length - a.d.window) : 0);
          bottom = min(bottom, sees);
          if (sees > mine) mine = sees, table_row = row;
        }
        w.max_low = __reduce_max_sync(0xffffffffu, top);
        w.min_high = __reduce_min_sync(0xffffffffu, bottom);
        const int most = w.end = __reduce_max_sync(0xffffffffu, mine);
        w.table_row = __shfl_sync(0xffffffffu, table_row, __ffs(__ballot_sync(0xffffffffu, mine == most)) - 1);
        const int all = (a.d.shared + kKeys - 1) / kKeys;
        const int per = (all + a.d.splits - 1) / a.d.splits;
        const int t0 = min(all, split * per), t1 = min((most + kKeys - 1) / kKeys, t0 + per);
        w.first = t0 * kKeys;
        w.tiles = max(0, t1 - t0);
        w.n[0] = alternate ? (w.tiles + 1) / 2 : w.tiles;
        w.n[1] = kUnits == 1 ? 0 : alternate ? w.tiles / 2 : w.tiles;
      }
      if (w.stop >= 0) {
        const int at = items % kItems;
        if (items >= kItems && !(ok = wait(sh, a.wait_limit, sh.item_empty[at], (items / kItems - 1) & 1))) break;
        if (lane == 0) {
          sh.item[at] = w;
          mbar_arrive(smem_u32(&sh.item_full[at]));
        }
        __syncwarp();
        items++;
        if (w.stop) break;
      }
      if (kPacked) {
        if (w.stop == 0 && !(ok = wait_item(sh, a.wait_limit, sh.want, (items - 1) & 1))) break;
        if (lane == 0) {
          fence_async_smem();  // the last answer has been read
          mbar_expect_tx(smem_u32(&sh.next_block), 16);
          take_block(smem_u32(&sh.answer), smem_u32(&sh.next_block));
          sh.asked = asks + 1;
        }
        asks++;
        if (!(ok = wait(sh, a.wait_limit, sh.next_block, (asks - 1) & 1))) break;
        block = taken_block(smem_u32(&sh.answer));
        __syncwarp();
      }
      }
      if (!ok && asks > 0) mbar_wait(smem_u32(&sh.next_block), (asks - 1) & 1);
    } else {
      // ---- loads, products and clean-up go through the tiles of every item
      const uint32_t lead = elect_one();
      const uint32_t columns = uniform(tmem);
      const int unit = warp >= Cfg::kOWarp ? warp - Cfg::kOWarp : warp - Cfg::kSWarp;  // of products
      Ring place;
      int q_uses = 0, number = 0;  // items with tiles; products of this warp
      for (int items = 0; ok; items++) {
        const int at = items % kItems;
        if (!(ok = wait_item(sh, a.wait_limit, sh.item_full[at], (items / kItems) & 1))) break;
        const Item &w = sh.item[at];
        if (uniform(w.stop)) break;
        const int tiles = uniform(w.tiles), alternate = MODE == kTcPrompt ? 0 : uniform(w.alternate);
        if (warp == Cfg::kKWarp) {
          // ---- queries and keys
          if (tiles > 0) {
            if (q_uses > 0 && !(ok = wait(sh, a.wait_limit, sh.q_empty, (q_uses - 1) & 1))) break;
            if (lead) {
              const uint32_t bar = smem_u32(&sh.q_full);
              const int units = alternate ? 1 : kUnits;
              mbar_expect_tx(bar, units * DP / 64 * per_unit * 128);
              for (int u = 0; u < units; u++)
                for (int s = 0; s < DP / 64; s++)
                  tma_load_4d(base + u * Cfg::kQBytes + s * kUnitRows * 128, &q_map, s * 64, 0, w.kv_head,
                              w.q0 + w.token0 + u * a.tokens, bar);
            }
            __syncwarp();
            q_uses++;
          }
          ok = load_tiles<MODE, DP, false>(sh, w, tiles, a, &k_map, k_ring, lead, place);
          if (tiles == 0 && lead) mbar_arrive(smem_u32(&sh.want));
        } else if (warp == Cfg::kVWarp) {
          // ---- values
          ok = load_tiles<MODE, DP, true>(sh, w, tiles, a, &v_map, v_ring, lead, place);
        } else if (warp == Cfg::kScrubWarp || warp >= Cfg::kOWarp + kUnits) {
          // ---- values that are not finite leave mixed tiles; the others are passed on
          // rows behind the last key are no one's: other sequences, or what the ring held before
          const int keys = MODE == kTcPrompt ? w.lk : MODE == kTcShared ? a.d.shared : w.end;
          bool found = false;
          for (int t = 0; t < tiles && ok; t++) {
            const bool mix = mixed<MODE, kKeys>(w, t);
            for (int c = 0; c < kChunks; c++, place.next()) {
              if (!(ok = wait(sh, a.wait_limit, sh.v_full[place.slot], place.parity()))) break;
              if (mix) {
                const uint32_t v = v_ring + place.slot * Cfg::kChunkBytes;
                // an exponent of all ones carries into the sign's place
                constexpr uint32_t kExp = BF16 ? 0x7f807f80u : 0x7c007c00u;
                constexpr uint32_t kOne = BF16 ? 0x00800080u : 0x04000400u;
                const int who = warp == Cfg::kScrubWarp ? 0 : warp - (Cfg::kOWarp + kUnits) + 1;
                constexpr int kStep = 32 * Cfg::kScrubWarps;
                uint32_t any = 0;
#pragma unroll 8
                for (int j = who * 32 + lane; j < Cfg::kChunkBytes / 16; j += kStep) {
                  const uint4 x = lds16(v + j * 16);
                  any |= ((x.x & kExp) + kOne) | ((x.y & kExp) + kOne) | ((x.z & kExp) + kOne) | ((x.w & kExp) + kOne);
                }
                if (any & 0x80008000u) {
                  for (int j = who * 32 + lane; j < Cfg::kChunkBytes / 16; j += kStep) {
                    const uint4 x = lds16(v + j * 16);
                    bool bad = false;
                    uint32_t y[4] = {x.x, x.y, x.z, x.w};
                    for (int k = 0; k < 4; k++) y[k] = zero_not_finite<BF16>(y[k], bad);
                    if (!bad) continue;
                    found |= key_of<MODE, kKeys>(w, t) + c * Cfg::kVKeys + j / 8 % Cfg::kVKeys < keys;
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(v + j * 16), "r"(y[0]),
                                 "r"(y[1]), "r"(y[2]), "r"(y[3])
                                 : "memory");
                  }
                }
                if (found) sh.item[at].wild = 1;
                fence_async_smem();
                __syncwarp();
              }
              if (lead) mbar_arrive(smem_u32(&sh.v_clean[place.slot]));
            }
          }
        } else if (warp < Cfg::kOWarp) {
          // ---- products S of one unit. Tiles that are not its own are given back at once.
          constexpr uint32_t kQk = idesc(BF16, kKeys, false);
          constexpr int kQSlab = kUnitRows * 128, kKSlab = kKeys * 128;
          const uint64_t qd = sw128_desc(base + (alternate ? 0 : unit) * Cfg::kQBytes);
          const int n = uniform(w.n[unit]);
          if (tiles > 0 && !(ok = wait(sh, a.wait_limit, sh.q_full, q_uses++ & 1))) break;
          if (tiles > 0 && n == 0 && lead) mbar_arrive(smem_u32(&sh.q_empty));
          for (int t = 0, left = n; t < tiles && ok; t++) {
            const bool mine = is_mine(alternate, unit, t, n);
            if (mine && number > 0 && !(ok = wait(sh, a.wait_limit, sh.s_free[unit], (number - 1) & 1)))
              break;  // S has been read
#pragma unroll
            for (int c = 0; c < kChunks; c++, place.next()) {
              if (!(ok = wait(sh, a.wait_limit, sh.k_full[place.slot], place.parity()))) break;
              const uint32_t empty = smem_u32(&sh.k_empty[place.slot]);
              if (!mine) {
                if (lead) mbar_arrive(empty);
                continue;
              }
              fence_after();
              const uint64_t kd = sw128_desc(k_ring + place.slot * Cfg::kChunkBytes);
#pragma unroll
              for (int k = 0; k < 4 * Cfg::kKSlabs; k++)
                mma_ss_if(lead, columns + unit * Cfg::kUnitCols,
                          qd + ((c * Cfg::kKSlabs + k / 4) * kQSlab >> 4) + (k % 4) * 2,
                          kd + ((k / 4) * kKSlab >> 4) + (k % 4) * 2, kQk, c > 0 || k > 0);
              if (c == kChunks - 1) commit_if(lead, smem_u32(&sh.s_full[unit]));
              commit_if(lead, empty);
            }
            if (!mine || !ok) continue;
            if (--left == 0) commit_if(lead, smem_u32(&sh.q_empty));  // the queries have been read
            number++;
          }
        } else {
          // ---- products O of one unit
          constexpr uint32_t kPv = idesc(BF16, DP, true);
          constexpr int kVSlab = Cfg::kVKeys * 128;
          const int n = uniform(w.n[unit]);
          const uint32_t d = columns + Cfg::kOCol + unit * DP;
          for (int t = 0, own = 0; t < tiles && ok; t++) {
            const bool mine = is_mine(alternate, unit, t, n);
            const int which = p_of(unit, number);
            const uint32_t p = columns + unit * Cfg::kUnitCols + Cfg::kPCol + (which - unit) * kKeys / 2;
            if (mine && !(ok = wait(sh, a.wait_limit, sh.p_full[which], p_round(number) & 1))) break;
#pragma unroll
            for (int c = 0; c < kChunks; c++, place.next()) {
              if (!(ok = wait(sh, a.wait_limit, sh.v_clean[place.slot], place.parity()))) break;
              const uint32_t empty = smem_u32(&sh.v_empty[place.slot]);
              if (!mine) {
                if (lead) mbar_arrive(empty);
                continue;
              }
              fence_after();
              const uint64_t vd = v_desc(v_ring + place.slot * Cfg::kChunkBytes, kVSlab);
#pragma unroll
              for (int k = 0; k < Cfg::kVKeys / 16; k++)
                mma_ts_if(lead, d, p + (c * Cfg::kVKeys / 16 + k) * 8, vd + k * (2048 >> 4), kPv,
                          own > 0 || c > 0 || k > 0);
              if (c == kChunks - 1) commit_if(lead, smem_u32(&sh.pv_done[which]));
              commit_if(lead, empty);
            }
            if (mine) number++, own++;
          }
        }
        __syncwarp();
        if (ok && lead) mbar_arrive(smem_u32(&sh.item_empty[at]));
      }
      if (!ok) {  // copies and products in flight end before the block does
        if (warp >= Cfg::kSWarp && warp < Cfg::kOWarp + kUnits) {
          uint64_t &bar = sh.drain[warp - Cfg::kSWarp];
          commit_if(lead, smem_u32(&bar));
          mbar_wait(smem_u32(&bar), 0);
        } else if (warp == Cfg::kKWarp || warp == Cfg::kVWarp) {
          const int issued = (int)min((uint32_t)kSlots, place.round * kSlots + place.slot);
          place.back(issued);
          for (int i = 0; i < issued; i++, place.next())
            mbar_wait(smem_u32(warp == Cfg::kKWarp ? &sh.k_full[place.slot] : &sh.v_full[place.slot]), place.parity());
          if (warp == Cfg::kKWarp && q_uses > 0) mbar_wait(smem_u32(&sh.q_full), (q_uses - 1) & 1);
        }
      }
    }
  } else {
    // ---- softmax: one thread per row and side
    take_registers<Cfg::kSoftRegs>();
    const int unit = kSides == 1 ? warp >> 2 : 0, side = kSides == 1 ? 0 : warp >> 2, row = tid & 127;
    constexpr int kCols = kKeys / kSides, kDims = DP / kSides;  // of a thread
    // What the other thread of the row says; false where it has given up.
    const int voice = kSides == 2 ? side : unit;
    uint32_t talks = 0;
    auto swap_words = [&](float mine, float *theirs) -> bool {
      uint64_t &told = sh.told[warp & 3], &heard = sh.heard[warp & 3];
      if (talks > 0 && !wait(sh, a.wait_limit, heard, (talks - 1) & 1)) return false;
      sh.word[voice][row] = mine;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&told));
      if (!wait(sh, a.wait_limit, told, talks & 1)) return false;
      *theirs = sh.word[voice ^ 1][row];
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&heard));
      talks++;
      return true;
    };
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // TMEM lane of the warp's first row
    const uint32_t o_at = tmem + lanes + Cfg::kOCol + unit * DP;
    const float c = kPacked ? a.p.scale : a.d.scale;
    const int sinks = MODE == kTcChunks && a.p.window ? a.p.sinks : 0;
    const uint64_t cc = pair(c, c);
    constexpr float kRoom = kTileHeadroom<BF16>;
    constexpr int kScaled = Cfg::kScaled;
    const int dim = MODE == kTcPrompt ? a.p.dim : a.c.head_dim;
    int number = 0, others = 0;  // tiles of this unit so far, and of the other one
    for (int items = 0; ok; items++) {
      const int at = items % kItems;
      if (!(ok = wait_item(sh, a.wait_limit, sh.item_full[at], (items / kItems) & 1))) break;
      const Item &w = sh.item[at];
      if (w.stop) break;
      const int n = w.n[unit], alternate = MODE == kTcPrompt ? 0 : w.alternate;
      int low = 0, high = INT32_MAX;  // the keys that the row sees; all, if it is not in use
      int64_t out_at = 0, index = 0;
      const int token = w.token0 + (alternate ? 0 : unit * a.tokens) + row / group;
      const int head = w.kv_head * group + row % group;
      const bool valid = row < per_unit && token < (kPacked ? w.lq : a.d.batch);
      if (valid) {
        const int64_t r = w.q0 + (int64_t)token;
        if (kPacked) {
          low = low_of(a.p, w.lq, w.lk, token), high = high_of(a.p, w.lq, w.lk, token);
          out_at = r * a.p.out_stride[0] + head * a.p.out_stride[1];
          index = r * a.p.heads + head;
        } else {
          int length;
          sequence_of(a.c, a.d, token, &length);
          low = a.d.window ? max(0, length - a.d.window) : 0;
          high = min(length, a.d.shared);
          out_at = r * a.d.out_stride[0] + head * a.d.out_stride[1];
          index = r * a.d.heads + head;
        }
      }
      float m = -INFINITY, l = 0.0f;  // m in units of the raw score
      for (int i = 0; i < n; i++, number++) {
        if (!(ok = wait(sh, a.wait_limit, sh.s_full[unit], number & 1))) break;
        fence_after();
        const uint32_t s_at = tmem + lanes + unit * Cfg::kUnitCols;
        const int key = key_of<MODE, kKeys>(w, tile_of(alternate, unit, i)) + side * kCols;
        float x[kCols];
#pragma unroll
        for (int j = 0; j + 32 <= kCols; j += 32) tmem_ld32(s_at + side * kCols + j, x + j);
        if (kCols % 32) tmem_ld16(s_at + kCols / 32 * 32, reinterpret_cast<uint32_t *>(x + kCols / 32 * 32));
        tmem_wait_ld();
        fence_before();
        if (lane == 0) mbar_arrive(smem_u32(&sh.s_free[unit]));
        const int from = low - key, to = high - key;  // columns [from, to) are visible
        if (__any_sync(0xffffffffu, from > 0 || to < kCols)) {
          if (MODE == kTcChunks && key < sinks) {
            const int first = sinks - key;
#pragma unroll
            for (int j = 0; j < kCols; j++) x[j] = (j >= from || j < first) && j < to ? x[j] : -INFINITY;
          } else {
#pragma unroll
            for (int j = 0; j < kCols; j++) x[j] = j >= from && j < to ? x[j] : -INFINITY;
          }
        }
        float top[4] = {m, m, m, m};
#pragma unroll
        for (int j = 0; j < kCols; j += 8)
#pragma unroll
          for (int k = 0; k < 4; k++) top[k] = max3(top[k], x[j + 2 * k], x[j + 2 * k + 1]);
        float now = max3(top[0], top[1], fmaxf(top[2], top[3]));
        if (kSides == 2) {
          float other;
          if (!(ok = swap_words(now, &other))) break;
          now = fmaxf(now, other);
        }
        // 2^8: the slack of the running maximum. Each row goes by its own scores alone.
        const bool grows = (now - m) * c > 8.0f;
        if (__any_sync(0xffffffffu, grows)) {
          const float f = grows ? exp2_fast((m - now) * c) : 1.0f;
          if (i > 0) {
            if (!(ok = wait(sh, a.wait_limit, sh.pv_done[p_of(unit, number - 1)], p_round(number - 1) & 1))) break;
            fence_after();
#pragma unroll 1
            for (int j = side * kDims; j < (side + 1) * kDims; j += kScaled) {  // bound by the latency of its reads
              uint32_t o[kScaled];
#pragma unroll
              for (int k = 0; k < kScaled; k += 16) tmem_ld16(o_at + j + k, o + k);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < kScaled; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
#pragma unroll
              for (int k = 0; k < kScaled; k += 16) tmem_st16(o_at + j + k, o + k);
            }
          }
          l *= f;
          if (grows) m = now;
        }
        const float z = m == -INFINITY ? 0.0f : kRoom - m * c;
        const uint64_t zz = pair(z, z);
        // the last product that reads these columns is done
        const int which = p_of(unit, number), round = p_round(number);
        const uint32_t p_at = s_at + Cfg::kPCol + (which - unit) * kKeys / 2;
        if (round > 0) {
          if (!(ok = wait(sh, a.wait_limit, sh.pv_done[which], (round - 1) & 1))) break;
          fence_after();
        }
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < kCols; j += 16) {
          uint32_t p[8];
#pragma unroll
          for (int k = 0; k < 8; k++) {
            const uint64_t e = fma2(pair(x[j + 2 * k], x[j + 2 * k + 1]), cc, zz);
            const float e0 = exp2_fast(__uint_as_float((uint32_t)e));
            const float e1 = exp2_fast(__uint_as_float((uint32_t)(e >> 32)));
            sum[k & 1] = add2(sum[k & 1], pair(e0, e1));
            p[k] = pack2<BF16>(e0, e1);
          }
          tmem_st8(p_at + (side * kCols + j) / 2, p);
        }
        sum[0] = add2(sum[0], sum[1]);
        l += __uint_as_float((uint32_t)sum[0]) + __uint_as_float((uint32_t)(sum[0] >> 32));
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[which]));
      }
      if (!ok) break;
      // ---- result
      if (kSides == 2) {
        float other;
        if (!(ok = swap_words(l, &other))) break;
        l += other;
      }
      if (n > 0 && !(ok = wait(sh, a.wait_limit, sh.pv_done[p_of(unit, number - 1)], p_round(number - 1) & 1))) break;
      // Items whose tiles the units have taken in turn: each gives half of the dims, from both sums.
      const bool joins = kJoins && alternate;
      float f = 1.0f, f1 = 0.0f;  // of this unit's sum, and of the other's
      if (kJoins) others += w.n[unit ^ 1];
      if (joins) {
        float m1, l1;
        if (!(ok = swap_words(m, &m1)) || !(ok = swap_words(l, &l1))) break;
        // with its word the other has announced its last weights, so that one product is open at most
        if (!(ok = wait(sh, a.wait_limit, sh.pv_done[unit ^ 1], (others - 1) & 1))) break;
        const float top = fmaxf(m, m1);
        f = m == -INFINITY ? 0.0f : exp2_fast((m - top) * c);
        f1 = m1 == -INFINITY ? 0.0f : exp2_fast((m1 - top) * c);
        m = top;
        l = unit == 0 ? l * f + l1 * f1 : l1 * f1 + l * f;
      }
      fence_after();
      const bool wild = n > 0 && *(volatile int *)&sh.item[at].wild;
      const bool final = MODE == kTcPrompt || a.d.part.parts == 1;
      const int part = MODE == kTcChunks ? w.split : a.d.first_part + (alternate ? 2 * split + unit : split);
      const float inv = !final ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
      const int64_t part_at =
          MODE == kTcPrompt ? 0 : (int64_t)part * a.d.part.rows + index;
#pragma unroll 1
      for (int j = side * kDims + (joins ? unit * DP / 2 : 0); j < (joins ? (unit + 1) * DP / 2 : (side + 1) * kDims);
           j += 32) {
        float o[32];
        __syncwarp();
        if (joins) {
          float o1[32];
          tmem_ld32(o_at + j, o);
          tmem_ld32(tmem + lanes + Cfg::kOCol + (unit ^ 1) * DP + j, o1);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 32; k++) o[k] = o[k] * f + o1[k] * f1;
        } else if (n > 0) {
          tmem_ld32(o_at + j, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int k = 0; k < 32; k++) o[k] = 0.0f;
        }
        if (wild && valid) {  // rare: what was left out of the products
          for (int i = 0; i < (joins ? w.tiles : n); i++) {
            const int t = joins ? i : tile_of(alternate, unit, i), key = key_of<MODE, kKeys>(w, t);
            if (!mixed<MODE, kKeys>(w, t)) continue;
            for (int r = key < sinks ? key : max(key, low); r < min(key + kKeys, high); r++) {
              if (r < low && r >= sinks) continue;
              const uint16_t *v;
              if (MODE == kTcPrompt) {
                v = a.p.v + (w.k0 + (int64_t)r) * a.p.v_stride[0] + w.kv_head * a.p.v_stride[1];
              } else {
                const int page = a.c.table[(int64_t)w.table_row * a.c.max_pages + r / a.c.page_tokens];
                if ((unsigned)page >= (unsigned)a.c.pages) continue;
                v = reinterpret_cast<const uint16_t *>(
                        a.c.memory + page * a.c.page_bytes + a.d.layer * a.c.layer_bytes +
                        (a.c.kv_heads + w.kv_head) * a.c.head_bytes) +
                    (int64_t)(r % a.c.page_tokens) * dim;
              }
#pragma unroll
              for (int k = 0; k < 32; k += 8) {
                if (j + k >= dim) break;
                const uint4 x = *reinterpret_cast<const uint4 *>(v + j + k);
                const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 8; e++) {
                  const uint16_t h = (uint16_t)(y[e / 2] >> (16 * (e & 1)));
                  if (not_finite<BF16>(h)) o[k + e] += to_float<BF16>(h);
                }
              }
            }
          }
        }
        if (valid && final) {
          uint16_t *out = (kPacked ? a.p.out : a.d.out) + out_at + j;
          uint32_t h[16];
#pragma unroll
          for (int k = 0; k < 16; k++) h[k] = pack2<BF16>(o[2 * k] * inv, o[2 * k + 1] * inv);
#pragma unroll
          for (int k = 0; k < 32; k += 16) {
            if (j + k + 16 <= dim) store32(out + k, h + k / 2, a.wide);
            else if (j + k < dim)  // dim is a multiple of 8
              *reinterpret_cast<uint4 *>(out + k) = make_uint4(h[k / 2], h[k / 2 + 1], h[k / 2 + 2], h[k / 2 + 3]);
          }
        } else if (valid && l != 0.0f) {
          float *out = a.d.part.o + part_at * dim + j;
#pragma unroll
          for (int k = 0; k < 32; k += 8)
            if (j + k < dim) store32(out + k, reinterpret_cast<const uint32_t *>(o + k), a.wide);
        }
      }
      const bool speaks = side == 0 && !(joins && unit);
      if (valid && final && speaks) {
        float *lse = kPacked ? a.p.lse : a.d.lse;
        if (lse) lse[index] = l == 0.0f ? -INFINITY : (m * c - kRoom + log2_fast(l)) * kLn2;
      } else if (valid && speaks) {
        a.d.part.ml[part_at] = make_float2(m * c - kRoom, l);
      }
      fence_before();  // O has been read before the next item's weights are announced
      if (joins) {     // by both units
        float none;
        if (!(ok = swap_words(0.0f, &none))) break;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.item_empty[at]));
    }
    if (!ok) {  // stores to tensor memory end before it is freed
      __syncwarp();
      tmem_wait_st();
    }
  }
  fence_before();
  __syncthreads();
  if (tid == 0 && sh.abort) atomicExch(a.timeout, 1);
  if (warp == Cfg::kItemWarp) {
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

// K (which 0) or V (1) of a cache layer as {dim, token of a page, key/value head, page}
bool encode_cache(CUtensorMap *map, bool bf16, const KvView &c, int layer, int which, int rows) {
  const uint64_t dims[4] = {(uint64_t)c.head_dim, (uint64_t)c.page_tokens, (uint64_t)c.kv_heads, (uint64_t)c.pages};
  const int64_t strides[3] = {c.head_dim * 2, c.head_bytes, c.page_bytes};
  const uint32_t box[4] = {64, (uint32_t)rows, 1, 1};
  return encode(map, bf16, c.memory + layer * c.layer_bytes + which * c.kv_heads * c.head_bytes, 4, dims, strides, box);
}

template <int MODE, int DP, bool BF16>
int32_t launch(dim3 grid, const CUtensorMap *maps, const TcArgs &a, cudaStream_t s) {
  auto fn = tile_kernel<MODE, DP, BF16>;
  DM_CUDA(dm::ensure_smem_limit((const void *)fn), "attention shared memory");
  using Cfg = TcCfg<DP, kSidesOf<MODE, DP>>;
  return launch_chained("attention launch", fn, grid, Cfg::kThreads, Cfg::kSmem, s, maps[0],
                        maps[1], maps[2], a);
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
// keys of a tile, and of a chunk of V
int keys_of(int dim) { return dim > 64 && dim <= 128 ? TcCfg<128>::kKeys : TcCfg<64>::kKeys; }
int v_keys_of(int dim) { return dim > 128 ? TcCfg<256>::kVKeys : keys_of(dim); }

// a box lies in one page and divides a chunk: pages are powers of two from 16
void boxes(const KvView &c, TcArgs *a) {
  auto rows = [&](int keys) { return std::min(c.page_tokens, keys & -keys); };
  a->k_box = rows(keys_of(c.head_dim));
  a->v_box = rows(v_keys_of(c.head_dim));
}

bool aligned32(const uint16_t *p, const int64_t *stride) {
  return ((uintptr_t)p & 31) == 0 && stride[0] % 16 == 0 && stride[1] % 16 == 0;
}

}  // namespace

bool tile_prompt_fits(const PromptArgs &p) {
  // broadcast tensors (stride 0) go to blocks of 16 rows, as strides that no map holds
  for (const int64_t *s : {p.q_stride, p.k_stride, p.v_stride})
    if (s[0] <= 0 || s[1] <= 0 || s[0] >= (int64_t)1 << 37 || s[1] * p.group >= (int64_t)1 << 37) return false;
  return p.k_tokens > 0;
}

int64_t wait_limit(const dm_cuda_context *ctx) { return ctx->attention_wait ? ctx->attention_wait : kWaitCycles; }

int32_t launch_tile_prompt(int32_t type, const PromptArgs &p, dm_cuda_context *ctx, cudaStream_t stream) {
  TcArgs a{};
  a.p = p;
  a.tokens = kUnitRows / p.group;
  a.timeout = ctx->status + kStatusWord;
  a.wait_limit = wait_limit(ctx);
  const int64_t tiles = p.q_tokens / (units_of(p.dim) * a.tokens) + p.sequences;
  if (tiles * p.kv_heads > INT32_MAX) return fail(DM_ERR_OVERFLOW, "too many query rows");
  a.tiles = (int)tiles;
  a.wide = aligned32(p.out, p.out_stride);
  const bool bf16 = type == DM_BF16;
  CUtensorMap maps[3];
  const uint64_t dims[3] = {(uint64_t)p.dim, (uint64_t)p.kv_heads, (uint64_t)p.k_tokens};
  const uint32_t k_box[3] = {64, 1, (uint32_t)keys_of(p.dim)}, v_box[3] = {64, 1, (uint32_t)v_keys_of(p.dim)};
  const int64_t ks[2] = {p.k_stride[1] * 2, p.k_stride[0] * 2}, vs[2] = {p.v_stride[1] * 2, p.v_stride[0] * 2};
  if (!encode_q(&maps[0], bf16, p.q, p.q_stride, p.dim, p.group, p.kv_heads, p.q_tokens, a.tokens) ||
      !encode(&maps[1], bf16, p.k, 3, dims, ks, k_box) || !encode(&maps[2], bf16, p.v, 3, dims, vs, v_box))
    return fail(DM_ERR_COMMAND, "could not describe the attention tensors for TMA");
  return launch<kTcPrompt>(bf16, p.dim, dim3((unsigned)(tiles * p.kv_heads)), maps, a, stream);
}

bool tile_queries_fit(const int64_t *q_stride, int group) {  // as above: the cache has no strides of its own
  return q_stride[0] > 0 && q_stride[1] > 0 && q_stride[0] < (int64_t)1 << 37 && q_stride[1] * group < (int64_t)1 << 37;
}

int tile_chunk_tokens(int dim, int group) { return units_of(dim) * (kUnitRows / group); }

int32_t launch_tile_chunks(int32_t type, const PromptArgs &p, const DecodeArgs &d, const KvView &c,
                           cudaStream_t stream) {
  TcArgs a{};
  a.p = p;
  a.d = d;
  a.c = c;
  a.tokens = kUnitRows / p.group;
  a.timeout = d.timeout;
  a.wait_limit = d.wait_limit;
  const int64_t tiles = chunk_tiles(p.q_tokens, p.sequences, 1, tile_chunk_tokens(p.dim, p.group));
  if (tiles * p.kv_heads * d.splits > INT32_MAX) return fail(DM_ERR_OVERFLOW, "too many query rows");
  a.tiles = (int)tiles;
  a.wide = d.part.parts > 1 ? ((uintptr_t)d.part.o & 31) == 0 : aligned32(p.out, p.out_stride);
  const bool bf16 = type == DM_BF16;
  CUtensorMap maps[3];
  boxes(c, &a);
  if (!encode_q(&maps[0], bf16, p.q, p.q_stride, p.dim, p.group, p.kv_heads, p.q_tokens, a.tokens) ||
      !encode_cache(&maps[1], bf16, c, d.layer, 0, a.k_box) || !encode_cache(&maps[2], bf16, c, d.layer, 1, a.v_box))
    return fail(DM_ERR_COMMAND, "could not describe the cache for TMA");
  return launch<kTcChunks>(bf16, p.dim, dim3((unsigned)(tiles * p.kv_heads * d.splits)), maps, a, stream);
}

bool tile_shared_alternates(int dim, int group, int batch) {
  return units_of(dim) == 2 && batch <= kUnitRows / group;
}

bool describe_chunks(int32_t type, const KvView &c, int layer, int rows, CUtensorMap *maps) {
  return encode_cache(&maps[0], type == DM_BF16, c, layer, 0, rows) &&
         encode_cache(&maps[1], type == DM_BF16, c, layer, 1, rows);
}

bool describe_queries(int32_t type, const void *q, const int64_t *stride, int dim, int group, int kv_heads,
                      int64_t tokens, int box_tokens, CUtensorMap *map) {
  return encode_q(map, type == DM_BF16, q, stride, dim, group, kv_heads, tokens, box_tokens);
}

bool describe_keys(int32_t type, const KvView &c, int layer, int rows, CUtensorMap *map) {
  return encode_cache(map, type == DM_BF16, c, layer, 0, rows);
}

int tile_keys(int dim) { return keys_of(dim); }

int tile_shared_items(int dim, int kv_heads, int group, int batch) {
  const int units = tile_shared_alternates(dim, group, batch) ? 1 : units_of(dim);
  const int per = units * (kUnitRows / group);
  return kv_heads * ((batch + per - 1) / per);
}

int32_t launch_tile_shared(int32_t type, const DecodeArgs &d, const KvView &c, cudaStream_t stream) {
  TcArgs a{};
  a.d = d;
  a.c = c;
  a.tokens = kUnitRows / d.group;
  a.alternate = tile_shared_alternates(c.head_dim, d.group, d.batch);
  a.timeout = d.timeout;
  a.wait_limit = d.wait_limit;
  a.wide = d.part.parts > 1 ? ((uintptr_t)d.part.o & 31) == 0 : aligned32(d.out, d.out_stride);
  const bool bf16 = type == DM_BF16;
  CUtensorMap maps[3];
  boxes(c, &a);
  if (!encode_q(&maps[0], bf16, d.q, d.q_stride, c.head_dim, d.group, c.kv_heads, d.batch, a.tokens) ||
      !encode_cache(&maps[1], bf16, c, d.layer, 0, a.k_box) || !encode_cache(&maps[2], bf16, c, d.layer, 1, a.v_box))
    return fail(DM_ERR_COMMAND, "could not describe the cache for TMA");
  const int items = tile_shared_items(c.head_dim, c.kv_heads, d.group, d.batch);
  return launch<kTcShared>(bf16, c.head_dim, dim3((unsigned)items, (unsigned)d.splits), maps, a, stream);
}

}  // namespace dma

extern "C" int32_t dm_selftest_attention_wait(dm_cuda_context *ctx, int64_t cycles) {
  if (!ctx) return fail(DM_ERR_INVALID_ARGUMENT, "null context");
  if (cycles < 0 || cycles > dm::tc::kWaitCycles)
    return fail(DM_ERR_INVALID_ARGUMENT, "the wait limit must be 1..%lld cycles, or 0", dm::tc::kWaitCycles);
  ctx->attention_wait = cycles;
  return DM_OK;
}

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
