// dm_attention.cuh -- shared parts of the attention kernels (include/diskmule_attention.h).
//
// All of them keep, per query row, a reference m (the running maximum of the scores times
// log2 e, less a constant for f16), the sum l of 2^(score - m) and the output sum o of
// 2^(score - m) v, in f32. Two such states over disjoint keys join as m = max(m1, m2),
// l = l1 2^(m1 - m) + l2 2^(m2 - m), o likewise, whatever their references are; the result is
// o / l and lse = (m + log2 l) ln 2.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "dm_kvcache.cuh"

namespace dma {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kStatusWord = 48;  // of the context's status buffer: a bounded wait ran out
constexpr float kLn2 = 0.6931471805599453f;

struct PromptArgs {
  const uint16_t *q, *k, *v;
  uint16_t *out;
  float *lse;
  int64_t q_stride[2], k_stride[2], v_stride[2], out_stride[2];
  const int32_t *q_offsets, *k_offsets;
  int64_t q_tokens, k_tokens;
  int32_t heads, kv_heads, group, dim, sequences, causal, window;
  int32_t sinks;  // chunks: with a window, keys below this are seen all the same
  float scale;    // times log2 e
};

// States of parts of the keys: o [part][row][dim], ml [part][row] = (m, l), with row =
// batch * heads + head. o is undefined where l is zero.
struct PartArgs {
  float *o;
  float2 *ml;
  int32_t parts;
  int64_t rows;
};

// Token i of lq stands at key place_of(); it sees the keys [low_of(), high_of()). Lengths and
// window may be anything up to 2^31, so no sum may exceed the larger of its terms.
__device__ __forceinline__ int place_of(int lq, int lk, int i) { return i - lq + lk; }
__device__ __forceinline__ int low_of(const PromptArgs &p, int lq, int lk, int i) {
  return p.window ? max(0, max(0, place_of(lq, lk, i)) - (p.window - 1)) : 0;
}
__device__ __forceinline__ int high_of(const PromptArgs &p, int lq, int lk, int i) {
  return p.causal ? max(0, min(lk, place_of(lq, lk, i) + 1)) : lk;
}

// Decode; of chunks the parts, the cache's side and the waits.
struct DecodeArgs {
  const uint16_t *q;
  uint16_t *out;
  float *lse;
  int64_t q_stride[2], out_stride[2];
  const int32_t *sequences;
  int32_t heads, group, batch, layer, window, shared, max_length;
  float scale;
  PartArgs part;       // part.parts == 1: results go straight to out and lse
  int32_t first_part;  // of this launch
  int32_t splits;      // parts of this launch
  int32_t joins;       // own part: this launch joins the parts before its own
  int32_t *timeout;    // set when a bounded wait runs out
  int64_t wait_limit;  // clocks
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Weights are rounded to 16 bits for the product with V. f16 has its full precision from 2^-14
// to 2^16 only: with the largest weight at 1, keys whose weights lie below 2^-14 would lose
// bits and those below 2^-25 be gone, however many they are. So f16 weights are 2^(score -
// maximum + headroom), as large as the type takes: 2^15, and 2^7 on tiles, whose reference may
// lie 2^8 below the maximum. bf16 has the range of f32.
template <bool BF16>
constexpr float kRowsHeadroom = BF16 ? 0.0f : 15.0f;
template <bool BF16>
constexpr float kTileHeadroom = BF16 ? 0.0f : 7.0f;

// two f32 -> two 16-bit values, `low` in the low half
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float low, float high) {
  uint32_t r;
  if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
  return r;
}

// 32 bytes at once where `wide` (the address is a multiple of 32), else 16
__device__ __forceinline__ void store32(void *p, const uint32_t *r, bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4 *>(p)[0] = make_uint4(r[0], r[1], r[2], r[3]);
    reinterpret_cast<uint4 *>(p)[1] = make_uint4(r[4], r[5], r[6], r[7]);
  }
}

// 16-bit patterns whose exponent is all ones are infinities and NaN
template <bool BF16>
__device__ __forceinline__ bool not_finite(uint16_t x) {
  constexpr uint16_t e = BF16 ? 0x7f80 : 0x7c00;
  return (x & e) == e;
}
template <bool BF16>
__device__ __forceinline__ float to_float(uint16_t x) {
  if (BF16) return __uint_as_float((uint32_t)x << 16);
  return __half2float(__ushort_as_half(x));
}
// x with its non-finite halves zeroed; `any` is set where there are some
template <bool BF16>
__device__ __forceinline__ uint32_t zero_not_finite(uint32_t x, bool &any) {
  if (not_finite<BF16>((uint16_t)x)) x &= 0xffff0000u, any = true;
  if (not_finite<BF16>((uint16_t)(x >> 16))) x &= 0xffffu, any = true;
  return x;
}

// Packed prompts: sequence and place of tile `tile` when a sequence of L tokens has
// ceil(L * per_token / rows) tiles. One warp; seq = -1 behind the last tile, and then `behind`
// is how far.
struct TileOf {
  int seq, tile, q0, q1, k0, k1;  // query and key rows of the sequence
  int64_t behind;
};
__device__ __forceinline__ TileOf find_tile(const PromptArgs &p, int per_token, int rows, int64_t tile) {
  const int lane = threadIdx.x & 31;
  TileOf r{-1, 0, 0, 0, 0, 0, 0};
  for (int s0 = 0; s0 < p.sequences; s0 += 32) {
    const int s = s0 + lane;
    int q0 = 0, q1 = 0, k0 = 0, k1 = 0;
    if (s < p.sequences) {  // rows outside the tensors are not there
      q0 = p.q_offsets[s], q1 = p.q_offsets[s + 1], k0 = p.k_offsets[s], k1 = p.k_offsets[s + 1];
      q0 = (int)min((int64_t)max(q0, 0), p.q_tokens), q1 = max(q0, (int)min((int64_t)q1, p.q_tokens));
      k0 = (int)min((int64_t)max(k0, 0), p.k_tokens), k1 = max(k0, (int)min((int64_t)k1, p.k_tokens));
    }
    const int64_t n = ((int64_t)(q1 - q0) * per_token + rows - 1) / rows;
    int64_t upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += u;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, tile < upto);
    if (hit) {
      const int src = __ffs(hit) - 1;
      r.seq = s0 + src;
      r.tile = (int)__shfl_sync(0xffffffffu, tile - (upto - n), src);
      r.q0 = __shfl_sync(0xffffffffu, q0, src);
      r.q1 = __shfl_sync(0xffffffffu, q1, src);
      r.k0 = __shfl_sync(0xffffffffu, k0, src);
      r.k1 = __shfl_sync(0xffffffffu, k1, src);
      return r;
    }
    tile -= __shfl_sync(0xffffffffu, upto, 31);
  }
  r.behind = tile;
  return r;
}

// Chunks, where there may be many entries, and many without rows: entry s has the numbers from
// T(s) = q0 per_token / rows + min(s, q0) on, q0 being its first row. T grows by at least as many as an
// entry has tiles, whatever lies before it, and ends at chunk_tiles below; so the entry of a number is
// searched for, 32 places at a time, and some numbers have no tile (seq = -1). One warp. (A sum over
// the entries, as above, took a block 1 us for each 32 of them: 3 busy entries among 4096 3300 us,
// now 15.)
__device__ __forceinline__ TileOf find_sparse_tile(const PromptArgs &p, int per_token, int rows, int64_t tile) {
  const int lane = threadIdx.x & 31;
  TileOf r{-1, 0, 0, 0, 0, 0, 0};
  int low = 0, count = p.sequences;
  while (true) {
    const int step = (count + 31) / 32;
    const int64_t s = low + (int64_t)lane * step;
    int q0 = 0, q1 = 0;
    bool below = s < (int64_t)low + count;
    if (below) {  // rows outside the tensor are not there
      q0 = (int)min((int64_t)max(p.q_offsets[s], 0), p.q_tokens);
      q1 = max(q0, (int)min((int64_t)p.q_offsets[s + 1], p.q_tokens));
      below = (int64_t)q0 * per_token / rows + min(s, (int64_t)q0) <= tile;
    }
    const int hits = __popc(__ballot_sync(0xffffffffu, below));
    if (hits == 0) return r;
    const int end = low + count;
    low += (hits - 1) * step;
    if (step == 1) {
      r.q0 = __shfl_sync(0xffffffffu, q0, hits - 1);
      r.q1 = __shfl_sync(0xffffffffu, q1, hits - 1);
      break;
    }
    count = min(step, end - low);
  }
  const int64_t in = tile - ((int64_t)r.q0 * per_token / rows + min(low, r.q0));
  if (in * rows < (int64_t)(r.q1 - r.q0) * per_token) r.seq = low, r.tile = (int)in;
  return r;
}
// Numbers of tiles of `rows` rows that chunks of `tokens` rows in all take, per_token to a token.
inline int64_t chunk_tiles(int64_t tokens, int sequences, int per_token, int rows) {
  return tokens * per_token / rows + std::min<int64_t>(sequences, tokens);
}

// Chunks: the keys that an item's rows see, [0, end) where the window reaches back to the sinks, else
// [0, sinks) and [low, end). Numbered without the gap they are [0, keys). sinks is a multiple of
// `unit`, so a run of `unit` numbers from a multiple of it on is a run of keys, and low is one of
// the power of two in `unit`, so that boxes of that size lie in one page.
struct Range {
  int sinks, low, keys;
  __device__ __forceinline__ int key(int number) const { return number < sinks ? number : number - sinks + low; }
};
__device__ __forceinline__ Range range_of(const PromptArgs &p, int low, int end, int unit) {
  Range r{0, 0, end};
  // no end is near 2^31, and sinks beyond it are all there are
  const int sinks = p.window ? (min(p.sinks, end) + unit - 1) / unit * unit : 0;
  low = low / (unit & -unit) * (unit & -unit);
  if (low > sinks) r = Range{sinks, low, sinks + max(0, end - low)};
  return r;
}

// Row of the page table and tokens of batch entry b; an entry that is out of range is empty.
__device__ __forceinline__ int sequence_of(const KvView &c, const DecodeArgs &a, int b, int *length) {
  const int row = a.sequences ? a.sequences[b] : b;
  if (row < 0 || row >= c.max_sequences) {
    *length = 0;
    return 0;
  }
  *length = min(max(c.lengths[row], 0), min(a.max_length, c.max_pages * c.page_tokens));
  return row;
}

// Strides of a call, {token, head} (both 0: contiguous), and the scale of its scores.
int32_t check_strides(const int64_t *given, int64_t heads, int dim, int64_t *use, const char *what);
int32_t check_scale(float given, int dim, float *use);

}  // namespace dma
