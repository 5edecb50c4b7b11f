// dm_rotate.cu -- norms of each head and position rotation, on the way from the projections to
// the queries and into the paged cache (include/diskmule_attention.h).
//
// A head's values x become w x / sqrt(mean x^2 + epsilon), and pairs (a, b) of them then
// (a cos t - b sin t, a sin t + b cos t) with t = position * frequency. Positions may be in the
// millions, where an f32 angle has lost its fraction of a turn; so frequencies are kept in turns
// per position as fractions of 2^64, the product with the position wraps around exactly where
// whole turns do, and its upper 32 bits are the angle. (Its f32, for the sines, is off by up to 2^-26
// of a turn; all else is below 2^-32 of one.)
//
// A warp takes a token. 8, 16 or 32 lanes hold a head, 16 bytes a lane: the sum of squares is a
// few shuffles, and a pair's other half is another lane's vector. Sines and weights are multiplied
// once for all heads of a token, and the next heads are on their way while some are done.
//
// 8191 tokens of 32 + 8 + 8 heads of dim 128 (201 MB) take 42 us, 4.8 TB/s of a copy's 6.5; the same
// loads and stores alone take 33. No unit is near its limit (DRAM 46% busy, issue 58%): it is the
// latency of a token's look-ups (entry, length, page, positions) and sines, a chain of 2 to 3 us, and
// of its heads behind them, which 28 warps an SM hide in part: 3802 tokens of 16 + 2 + 2 heads of dim
// 256 (78 MB) 19 us. (One block for eight tokens with the sines in shared
// memory 94 and 51 us; loads through a ring in shared memory 51 and 33, four at a time in registers
// and 16 warps 49 and 29.) Few tokens are latency: 5 us.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <new>

#include "dm_attention.cuh"

using dmi::fail;

struct dm_rope {
  dm_cuda_context *ctx = nullptr;
  int32_t rotary_dim = 0, interleaved = 0, axes = 1;
  float scale = 1.0f;
  uint64_t *turns = nullptr;     // device [rotary_dim / 2]: of each pair per position, in 2^-64
  int32_t *pair_axes = nullptr;  // device, behind them
};

namespace dma {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kBlocks = 7;   // of an SM
constexpr int kPairs = 128;  // at most
constexpr int kFlight = 2;   // 16-byte loads of a thread in flight

enum Kind { kQ, kK, kV };

struct RotateArgs {
  const uint8_t *in[3];
  uint8_t *out[3];                          // null: not wanted
  int64_t in_stride[3][2], out_stride[3][2];  // [token, head], bytes
  const float *weight[2];
  const int32_t *positions, *rows, *offsets;
  const uint64_t *turns;
  const int32_t *pair_axes;
  int64_t tokens;
  int32_t first[3], heads;  // first row of each kind among a token's; rows of a token
  int32_t dim, rotary, interleaved, norms, sequences, layer, cached;
  float scale, epsilon;
};

// The entry that owns row t, or -1: the last whose offset is not above it, if its end is. One warp.
__device__ __forceinline__ int entry_of(const int32_t *offsets, int n, int64_t t) {
  const int lane = threadIdx.x & 31;
  int low = 0, count = n;
  while (count > 0) {
    const int step = (count + 31) / 32;
    const int64_t at = low + (int64_t)lane * step;
    const bool below = at < (int64_t)low + count && offsets[at] <= t;
    const int hits = __popc(__ballot_sync(0xffffffffu, below));
    if (hits == 0) return -1;
    const int end = low + count;
    low += (hits - 1) * step;
    if (step == 1) break;
    count = min(step, end - low);
  }
  return n > 0 && t < offsets[low + 1] ? low : -1;
}

// Two 16-bit values as f32
template <bool BF16>
__device__ __forceinline__ float2 both(uint32_t x) {
  if (BF16) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2 *>(&x));
}

__device__ __forceinline__ float rsqrt_fast(float x) {  // within two units of the last place
  float y;
  asm("rsqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Values of a head that one lane has, as pairs of f32
struct Eight {
  float2 v[4];
};
template <bool BF16>
__device__ __forceinline__ Eight unpack(const uint32_t *r) {
  return Eight{{both<BF16>(r[0]), both<BF16>(r[1]), both<BF16>(r[2]), both<BF16>(r[3])}};
}

// Warp (x, warp) does part y of a token's heads.
template <int LANES, bool BF16>
__global__ void __launch_bounds__(kThreads, kBlocks) rotate_kernel(const __grid_constant__ KvView c,
                                                                   const __grid_constant__ RotateArgs a) {
  constexpr unsigned kAll = 0xffffffffu;
  constexpr int kSide = 32 / LANES;  // heads side by side
  __shared__ alignas(16) float cosine[kWarps][LANES * 8], sine[kWarps][LANES * 8];  // of each value of the token's heads
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int vec = lane % LANES, side = lane / LANES, col = vec * 8;
  const int64_t t = (int64_t)blockIdx.x * kWarps + warp;
  if (t >= a.tokens) return;
  const bool in = col < a.dim;
  const int begin = (int)((int64_t)a.heads * blockIdx.y / gridDim.y);
  const int end = (int)((int64_t)a.heads * (blockIdx.y + 1) / gridDim.y);
  wait_for_previous();
  let_next_start();

  // Heads of a kind go kSide at a time, kFlight times as many to a batch; the next batch is on its
  // way while one is done.
  auto low_of = [&](int kind) { return max(begin, a.first[kind]); };
  auto high_of = [&](int kind) { return min(end, kind == kQ ? a.first[kK] : kind == kK ? a.first[kV] : a.heads); };
  int ahead = -1, left = -side;  // of the loads: kind, and heads from this lane's on
  const uint8_t *from = nullptr;
  int64_t from_step = 0;
  uint4 x[kFlight] = {};
  auto load = [&]() {
    while (left <= -side && ahead < kV) {
      ahead++;
      const int low = low_of(ahead);
      left = max(high_of(ahead) - low, 0) - side;
      from = a.in[ahead] + t * a.in_stride[ahead][0] + (low + side - a.first[ahead]) * a.in_stride[ahead][1] + col * 2;
      from_step = kSide * a.in_stride[ahead][1];
    }
#pragma unroll
    for (int k = 0; k < kFlight; k++, from += from_step)
      if (in && left > k * kSide) x[k] = *reinterpret_cast<const uint4 *>(from);
    left -= kFlight * kSide;
  };
  load();

  // ---- the token's place and its sines, while the first heads come in
  const int half = a.rotary / 2;
  uint64_t turns[kPairs / 32] = {};
  int64_t position[kPairs / 32] = {};
#pragma unroll
  for (int j = 0; j < kPairs / 32; j++)
    if (lane + 32 * j < half) {
      turns[j] = a.turns[lane + 32 * j];
      if (a.positions) position[j] = a.positions[a.pair_axes[lane + 32 * j] * a.tokens + t];
    }
  int64_t place = 0, cached_at = -1;
  const int page_bits = 31 - __clz(c.page_tokens);  // pages are powers of two
  if (a.cached) {
    const int i = entry_of(a.offsets, a.sequences, t);
    if (i < 0) return;
    const int row = a.rows ? a.rows[i] : i;
    int page = -1;
    if (row >= 0 && row < c.max_sequences) {
      const int length = c.lengths[row];
      place = length - ((int64_t)a.offsets[i + 1] - t);
      if (place >= 0 && place < length && (place >> page_bits) < c.max_pages)
        page = c.table[(int64_t)row * c.max_pages + (place >> page_bits)];
    }
    if ((unsigned)page < (unsigned)c.pages) {
      cached_at = page * c.page_bytes + a.layer * c.layer_bytes + (place & (c.page_tokens - 1)) * c.head_dim * 2 + col * 2;
    } else {
      place = 0;
      if (lane == 0 && blockIdx.y == 0) atomicOr(c.status, DM_KV_BAD_TOKEN);
    }
  }
#pragma unroll
  for (int j = 0; j < kPairs / 32; j++) {
    const int i = lane + 32 * j;
    if (i >= half) break;
    const uint64_t angle = (uint64_t)(a.positions ? position[j] : place) * turns[j];
    float s, k;
    // half turns, -1 to 1; their f32 is off by at most 2^-25
    sincospif((float)(int32_t)(angle >> 32) * 0x1p-31f, &s, &k);
    const int first = a.interleaved ? 2 * i : i, second = a.interleaved ? first + 1 : i + half;
    cosine[warp][first] = cosine[warp][second] = k * a.scale;
    sine[warp][first] = -s * a.scale;
    sine[warp][second] = s * a.scale;
  }
  __syncwarp();

  // where the other halves of this lane's pairs are; pairs side by side are exchanged in place
  const int other = a.interleaved || col >= a.rotary ? vec : col >= half ? vec - half / 8 : vec + half / 8;
  const float share = 1.0f / a.dim;
  Eight own{}, across{};  // a value is own times it plus across times the other of its pair, over the root
#pragma unroll 1
  for (int kind = kQ; kind <= kV; kind++) {
    const int n = high_of(kind) - low_of(kind), head = low_of(kind) + side - a.first[kind];
    if (n <= 0) continue;
    const bool normed = (a.norms >> kind) & 1, rotated = kind != kV && a.rotary > 0;
    const bool turning = rotated && col < a.rotary;
    if (kind != kV && in) {
      float k[8], s[8], here[8], there[8];
#pragma unroll
      for (int e = 0; e < 8; e++) k[e] = here[e] = there[e] = 1.0f, s[e] = 0.0f;
      auto fetch8 = [](const float *p, float *to) {
        const float4 u = reinterpret_cast<const float4 *>(p)[0], v = reinterpret_cast<const float4 *>(p)[1];
        to[0] = u.x, to[1] = u.y, to[2] = u.z, to[3] = u.w, to[4] = v.x, to[5] = v.y, to[6] = v.z, to[7] = v.w;
      };
      if (turning) fetch8(&cosine[warp][col], k), fetch8(&sine[warp][col], s);
      if (normed && a.weight[kind]) fetch8(a.weight[kind] + col, here), fetch8(a.weight[kind] + other * 8, there);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float x = a.interleaved ? there[e + 1] : there[e], y = a.interleaved ? there[e] : there[e + 1];
        own.v[e / 2] = make_float2(k[e] * here[e], k[e + 1] * here[e + 1]);
        across.v[e / 2] = make_float2(s[e] * x, s[e + 1] * y);
      }
    }
    const int64_t out_step = kSide * a.out_stride[kind][1], cache_step = kSide * c.head_bytes;
    const bool out_too = in && a.out[kind], cache_too = in && kind != kQ && cached_at >= 0;
    uint8_t *out = a.out[kind] + t * a.out_stride[kind][0] + head * a.out_stride[kind][1] + col * 2;
    uint8_t *cache = c.memory + cached_at + ((kind == kV ? c.kv_heads : 0) + head) * c.head_bytes;
#pragma unroll 1
    for (int i = 0; i < n; i += kFlight * kSide) {
      uint32_t r[kFlight][4];
#pragma unroll
      for (int k = 0; k < kFlight; k++) r[k][0] = x[k].x, r[k][1] = x[k].y, r[k][2] = x[k].z, r[k][3] = x[k].w;
      load();
      if (normed || rotated) {
        Eight v[kFlight];
        float root[kFlight];
#pragma unroll
        for (int k = 0; k < kFlight; k++) {
          v[k] = unpack<BF16>(r[k]);
          root[k] = 1.0f;
        }
        if (normed) {
#pragma unroll
          for (int k = 0; k < kFlight; k++) {
            float2 sum = __fmul2_rn(v[k].v[0], v[k].v[0]);
#pragma unroll
            for (int e = 1; e < 4; e++) sum = __ffma2_rn(v[k].v[e], v[k].v[e], sum);
            root[k] = in ? sum.x + sum.y : 0.0f;
          }
#pragma unroll
          for (int o = 1; o < LANES; o <<= 1)
#pragma unroll
            for (int k = 0; k < kFlight; k++) root[k] += __shfl_xor_sync(kAll, root[k], o);
#pragma unroll
          for (int k = 0; k < kFlight; k++) root[k] = rsqrt_fast(root[k] * share + a.epsilon);
        }
        if (kind != kV) {
          if (rotated)
#pragma unroll
            for (int k = 0; k < kFlight; k++)
#pragma unroll
              for (int e = 0; e < 4; e++)
                r[k][e] = a.interleaved ? __funnelshift_l(r[k][e], r[k][e], 16) : __shfl_sync(kAll, r[k][e], other, LANES);
#pragma unroll
          for (int k = 0; k < kFlight; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[k].v[e] = __fmul2_rn(v[k].v[e], own.v[e]);
          // what does not turn stays apart from the rest of its head: 0 times infinity is no zero
          if (turning)
#pragma unroll
            for (int k = 0; k < kFlight; k++) {
              const Eight u = unpack<BF16>(r[k]);
#pragma unroll
              for (int e = 0; e < 4; e++) v[k].v[e] = __ffma2_rn(u.v[e], across.v[e], v[k].v[e]);
            }
        }
#pragma unroll
        for (int k = 0; k < kFlight; k++) {
          const float2 scale = make_float2(root[k], root[k]);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float2 y = __fmul2_rn(v[k].v[e], scale);
            r[k][e] = pack2<BF16>(y.x, y.y);
          }
        }
      }
      if (out_too)
#pragma unroll
        for (int k = 0; k < kFlight; k++, out += out_step)
          if (i + k * kSide + side < n) *reinterpret_cast<uint4 *>(out) = make_uint4(r[k][0], r[k][1], r[k][2], r[k][3]);
      if (cache_too)
#pragma unroll
        for (int k = 0; k < kFlight; k++, cache += cache_step)
          if (i + k * kSide + side < n) *reinterpret_cast<uint4 *>(cache) = make_uint4(r[k][0], r[k][1], r[k][2], r[k][3]);
    }
  }
}

template <bool BF16>
int32_t launch_rotate(dim3 grid, cudaStream_t s, const KvView &c, const RotateArgs &a) {
  auto fn = a.dim <= 64 ? rotate_kernel<8, BF16> : a.dim <= 128 ? rotate_kernel<16, BF16> : rotate_kernel<32, BF16>;
  return launch_chained("rotate launch", fn, grid, kThreads, 0, s, c, a);
}

}  // namespace
}  // namespace dma

using namespace dma;

extern "C" {

int32_t dm_rope_create(dm_cuda_context *ctx, const dm_rope_desc *d, dm_rope **out) {
  if (!ctx || !d || !out) return fail(DM_ERR_INVALID_ARGUMENT, "null argument");
  *out = nullptr;
  if (d->rotary_dim <= 0 || d->rotary_dim % 16 || d->rotary_dim > 2 * kPairs)
    return fail(DM_ERR_ELEMENT_COUNT, "rotary_dim %d is not a multiple of 16 up to 256", d->rotary_dim);
  if (d->axes < 1 || d->axes > 4) return fail(DM_ERR_ELEMENT_COUNT, "%d axes of positions", d->axes);
  if (!std::isfinite(d->scale)) return fail(DM_ERR_NON_FINITE, "the scale of a rotation is not finite");
  if (!d->frequencies && !(std::isfinite(d->theta) && d->theta > 0.0))
    return fail(DM_ERR_POSITIVE_PARAMETER, "theta must be finite and positive");
  const int pairs = d->rotary_dim / 2;
  uint64_t turns[kPairs];
  int32_t axes[kPairs] = {};
  const long double whole = 2.0L * 3.141592653589793238462643383279502884L;
  for (int i = 0; i < pairs; i++) {
    const double f = d->frequencies ? d->frequencies[i] : std::pow(d->theta, -2.0 * i / d->rotary_dim);
    if (!std::isfinite(f)) return fail(DM_ERR_NON_FINITE, "frequency %d is not finite", i);
    long double t = f / whole;
    t -= floorl(t);  // whole turns a position leave no trace
    const long double u = ldexpl(t, 64);
    turns[i] = u >= 0x1p64L ? 0 : (uint64_t)u;
    if (d->pair_axes) axes[i] = d->pair_axes[i];
    if (axes[i] < 0 || axes[i] >= d->axes)
      return fail(DM_ERR_ELEMENT_COUNT, "pair %d turns with axis %d of %d", i, axes[i], d->axes);
  }
  dm_rope *r = new (std::nothrow) dm_rope;
  if (!r) return fail(DM_ERR_ALLOCATION, "could not allocate a rotation");
  cudaSetDevice(ctx->device);
  void *p = nullptr;
  if (cudaMalloc(&p, pairs * 12) != cudaSuccess) {
    cudaGetLastError();
    delete r;
    return fail(DM_ERR_ALLOCATION, "could not allocate %d bytes for a rotation", pairs * 12);
  }
  r->ctx = ctx;
  dmi::retain_context(ctx);
  r->rotary_dim = d->rotary_dim;
  r->interleaved = d->interleaved != 0;
  r->axes = d->axes;
  r->scale = d->scale == 0.0f ? 1.0f : d->scale;
  r->turns = (uint64_t *)p;
  r->pair_axes = (int32_t *)(r->turns + pairs);
  cudaError_t rc = cudaMemcpyAsync(r->turns, turns, pairs * 8, cudaMemcpyHostToDevice, ctx->stream);
  if (rc == cudaSuccess)
    rc = cudaMemcpyAsync(r->pair_axes, axes, pairs * 4, cudaMemcpyHostToDevice, ctx->stream);
  if (rc == cudaSuccess) rc = cudaStreamSynchronize(ctx->stream);
  if (rc != cudaSuccess) {
    dm_rope_destroy(r);
    return dmi::cuda_fail(rc, "rotation set-up");
  }
  *out = r;
  return DM_OK;
}

void dm_rope_destroy(dm_rope *r) {
  if (!r) return;
  cudaSetDevice(r->ctx->device);
  cudaFree(r->turns);
  dmi::release_context(r->ctx);
  delete r;
}

int32_t dm_attention_rotate(dm_cuda_context *ctx, const dm_rope *rope, dm_kv_cache *cache,
                            const dm_attention_rotate_desc *in, void *stream) {
  if (!ctx || !in) return fail(DM_ERR_INVALID_ARGUMENT, "null argument");
  if ((rope && rope->ctx != ctx) || (cache && cache->ctx != ctx))
    return fail(DM_ERR_INVALID_ARGUMENT, "the rotation or the cache belongs to another context");
  if (in->type != DM_BF16 && in->type != DM_F16)
    return fail(DM_ERR_UNSUPPORTED_TENSOR_TYPE, "rotation takes bf16 or f16");
  if (in->head_dim <= 0 || in->head_dim % 8 || in->head_dim > 256)
    return fail(DM_ERR_ELEMENT_COUNT, "head_dim %d is not a multiple of 8 up to 256", in->head_dim);
  if (rope && rope->rotary_dim > in->head_dim)
    return fail(DM_ERR_ELEMENT_COUNT, "%d values of %d turn", rope->rotary_dim, in->head_dim);
  if (in->norms & ~(DM_NORM_Q | DM_NORM_K | DM_NORM_V))
    return fail(DM_ERR_INVALID_ARGUMENT, "unknown norms %d", in->norms);
  if (in->norms && (!std::isfinite(in->epsilon) || in->epsilon < 0.0f))
    return fail(DM_ERR_POSITIVE_PARAMETER, "a norm needs a finite epsilon that is not negative");
  if (in->tokens < 0 || in->tokens > kMostTokens)
    return fail(DM_ERR_ELEMENT_COUNT, "a bad number of tokens");
  if (in->sequences < 0) return fail(DM_ERR_ELEMENT_COUNT, "%d sequences", in->sequences);
  const bool has[3] = {in->q != nullptr, in->k != nullptr, in->v != nullptr};
  if ((has[kQ] && (in->heads <= 0 || in->heads > 65535)) ||
      ((has[kK] || has[kV]) && (in->kv_heads <= 0 || in->kv_heads > 65535)))
    return fail(DM_ERR_ELEMENT_COUNT, "%d query and %d key/value heads", in->heads, in->kv_heads);
  const dm_kv_cache_desc *kd = cache ? &cache->desc : nullptr;
  if (cache) {
    if (kd->type != in->type || kd->head_dim != in->head_dim)
      return fail(DM_ERR_INVALID_ARGUMENT, "the cache has another type or head_dim");
    if (has[kK] != has[kV]) return fail(DM_ERR_INVALID_ARGUMENT, "a cache takes keys and values");
    if (has[kK] && kd->kv_heads != in->kv_heads)
      return fail(DM_ERR_ELEMENT_COUNT, "%d key/value heads, and the cache has %d", in->kv_heads, kd->kv_heads);
    if (in->layer < 0 || in->layer >= kd->layers)
      return fail(DM_ERR_INVALID_LAYER, "layer %d of %d", in->layer, kd->layers);
    if (in->sequences > kd->max_sequences)
      return fail(DM_ERR_ELEMENT_COUNT, "%d sequences, and the cache has %d", in->sequences, kd->max_sequences);
  }
  if (in->tokens == 0 || (cache && in->sequences == 0)) return DM_OK;
  if (cache && !in->offsets) return fail(DM_ERR_INVALID_ARGUMENT, "null offsets");
  if (!cache && rope && !in->positions && (has[kQ] || has[kK]))
    return fail(DM_ERR_INVALID_ARGUMENT, "without a cache a rotation needs positions");
  RotateArgs a{};
  const void *from[3] = {in->q, in->k, in->v};
  void *to[3] = {in->q_out, in->k_out, in->v_out};
  const int64_t *from_stride[3] = {in->q_stride, in->k_stride, in->v_stride};
  const int64_t *to_stride[3] = {in->q_out_stride, in->k_out_stride, in->v_out_stride};
  const char *names[3] = {"query", "key", "value"};
  for (int i = 0; i < 3; i++) {
    const int heads = i == kQ ? in->heads : in->kv_heads;
    a.first[i] = a.heads;
    if (to[i] && !has[i]) return fail(DM_ERR_INVALID_ARGUMENT, "a %s output without its input", names[i]);
    // what nobody receives is not read
    if (!has[i] || (!to[i] && (i == kQ || !cache))) continue;
    if (((uintptr_t)from[i] | (uintptr_t)to[i]) & 15)
      return fail(DM_ERR_INVALID_ARGUMENT, "rotated tensors must be 16-byte aligned");
    a.in[i] = (const uint8_t *)from[i];
    a.out[i] = (uint8_t *)to[i];
    if (int32_t rc = check_strides(from_stride[i], heads, in->head_dim, a.in_stride[i], names[i])) return rc;
    if (int32_t rc = check_strides(to_stride[i], heads, in->head_dim, a.out_stride[i], names[i])) return rc;
    // in place: else a token's result would lie where another warp is yet to read
    if (from[i] == to[i] && ((in->tokens > 1 && a.in_stride[i][0] != a.out_stride[i][0]) ||
                             (heads > 1 && a.in_stride[i][1] != a.out_stride[i][1])))
      return fail(DM_ERR_INVALID_ARGUMENT, "a %s rotated in place needs the same strides for its output", names[i]);
    for (int j = 0; j < 2; j++) a.in_stride[i][j] *= 2, a.out_stride[i][j] *= 2;
    a.heads += heads;
  }
  if (a.heads == 0) return DM_OK;
  if (((uintptr_t)in->q_weight | (uintptr_t)in->k_weight) & 15)
    return fail(DM_ERR_INVALID_ARGUMENT, "norm weights must be 16-byte aligned");
  a.weight[0] = in->q_weight;
  a.weight[1] = in->k_weight;
  a.positions = in->positions;
  a.rows = in->rows;
  a.offsets = in->offsets;
  a.tokens = in->tokens;
  a.dim = in->head_dim;
  a.norms = in->norms;
  a.epsilon = in->epsilon;
  a.sequences = in->sequences;
  a.layer = in->layer;
  a.cached = cache != nullptr;
  if (rope) {
    a.turns = rope->turns;
    a.pair_axes = rope->pair_axes;
    a.rotary = rope->rotary_dim;
    a.interleaved = rope->interleaved;
    a.scale = rope->scale;
  }
  cudaSetDevice(ctx->device);
  // A warp to a token; few tokens: their heads over several, down to two rounds each.
  const int side = a.dim <= 64 ? 4 : a.dim <= 128 ? 2 : 1;
  const int64_t blocks = (in->tokens + kWarps - 1) / kWarps;
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(148 * kBlocks / blocks, (a.heads + 2 * side - 1) / (2 * side)));
  const KvView view = cache ? cache->view : KvView{};
  const dim3 grid((unsigned)blocks, (unsigned)parts);
  return in->type == DM_BF16 ? launch_rotate<true>(grid, (cudaStream_t)stream, view, a)
                             : launch_rotate<false>(grid, (cudaStream_t)stream, view, a);
}

}  // extern "C"
