// dm_rotate.cu -- norms of each head and position rotation, on the way from the projections to
// the queries and into the paged cache (include/diskmule_attention.h).
//
// A head's values x become w x / sqrt(mean x^2 + epsilon), and pairs (a, b) of them then
// (a cos t - b sin t, a sin t + b cos t) with t = position * frequency. Positions may be in the
// millions, where an f32 angle has lost its fraction of a turn; so frequencies are kept in turns
// per position as fractions of 2^64, the product with the position wraps around exactly where
// whole turns do, and its upper 32 bits are the angle.
//
// A group of 8, 16 or 32 lanes holds one head, 16 bytes a lane: the sum of squares is a few
// shuffles, and a pair's other half is another lane's vector. A block computes the sines of its
// tokens once, for all their heads.
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

constexpr int kThreads = 256;
constexpr int kBlockTokens = 8;  // of a block at most: a warp looks after each
constexpr int kPairs = 128;
constexpr int kFlight = 4;      // loads of a thread in flight

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
  int32_t dim, rotary, interleaved, norms, sequences, layer, cached, block_tokens;
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

template <int LANES, bool BF16>
__global__ void __launch_bounds__(kThreads) rotate_kernel(const __grid_constant__ KvView c,
                                                          const __grid_constant__ RotateArgs a) {
  constexpr unsigned kAll = 0xffffffffu;
  constexpr int kGroups = kThreads / LANES;
  __shared__ float cosine[kBlockTokens][kPairs], sine[kBlockTokens][kPairs];
  __shared__ float weight[2][LANES * 8];
  __shared__ int64_t place_at[kBlockTokens];  // byte offset of the token's place in part 0 of its page; -1: none
  __shared__ int owned[kBlockTokens];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  wait_for_previous();
  let_next_start();

  for (int i = tid; i < 2 * LANES * 8; i += kThreads) {
    const int which = i / (LANES * 8), col = i % (LANES * 8);
    weight[which][col] = a.weight[which] && col < a.dim ? a.weight[which][col] : 1.0f;
  }
  const int64_t token0 = (int64_t)blockIdx.x * a.block_tokens;
  const int tokens = (int)min((int64_t)a.block_tokens, a.tokens - token0);
  if (warp < tokens) {
    const int64_t t = token0 + warp;
    int64_t place = 0;
    bool mine = true;
    if (a.cached) {
      const int i = entry_of(a.offsets, a.sequences, t);
      mine = i >= 0;
      if (mine) {
        const int row = a.rows ? a.rows[i] : i;
        int page = -1;
        if (row >= 0 && row < c.max_sequences) {
          const int length = c.lengths[row];
          place = length - ((int64_t)a.offsets[i + 1] - t);
          if (place >= 0 && place < length && place / c.page_tokens < c.max_pages)
            page = c.table[(int64_t)row * c.max_pages + place / c.page_tokens];
        }
        const bool fits = (unsigned)page < (unsigned)c.pages;
        if (lane == 0) {
          place_at[warp] = fits ? page * c.page_bytes + a.layer * c.layer_bytes +
                                      (place % c.page_tokens) * c.head_dim * 2 : -1;
          if (!fits && blockIdx.y == 0) atomicOr(c.status, DM_KV_BAD_TOKEN);
        }
        if (!fits) place = 0;
      }
    }
    if (lane == 0) owned[warp] = mine;
    if (mine)
      for (int i = lane; i < a.rotary / 2; i += 32) {
        const int64_t p = a.positions ? a.positions[a.pair_axes[i] * a.tokens + t] : place;
        const uint64_t turns = (uint64_t)p * a.turns[i];
        // half turns, -1 to 1; their f32 is off by at most 2^-25
        const float half = (float)(int32_t)(turns >> 32) * 0x1p-31f;
        float s, k;
        sincospif(half, &s, &k);
        cosine[warp][i] = k * a.scale;
        sine[warp][i] = s * a.scale;
      }
  }
  __syncthreads();

  const int group = tid / LANES, vec = tid % LANES, col = vec * 8;
  const int half = a.rotary / 2;
  const float share = 1.0f / a.dim;
  // where the other halves of this lane's pairs are
  const bool turns = col < a.rotary, upper = !a.interleaved && col >= half;
  const int other = turns && !a.interleaved ? (upper ? vec - half / 8 : vec + half / 8) : vec;
  const int pair0 = a.interleaved ? col / 2 : upper ? col - half : col;
  const int all = tokens * a.heads, stride = kGroups * gridDim.y;
  int at = blockIdx.y * kGroups + group;
  int token = at / a.heads, head = at % a.heads;
  // rounds are the same for all lanes of a warp
  for (int from = blockIdx.y * kGroups; from < all; from += kFlight * stride) {
    uint4 x[kFlight];
    int token_of[kFlight], head_of[kFlight];
    bool valid[kFlight];
#pragma unroll
    for (int k = 0; k < kFlight; k++) {
      token_of[k] = token, head_of[k] = head;
      valid[k] = at < all && col < a.dim && owned[min(token, kBlockTokens - 1)];
      x[k] = make_uint4(0, 0, 0, 0);
      if (valid[k]) {
        const int kind = head >= a.first[kV] ? kV : head >= a.first[kK] ? kK : kQ;
        x[k] = *reinterpret_cast<const uint4 *>(a.in[kind] + (token0 + token) * a.in_stride[kind][0] +
                                                (head - a.first[kind]) * a.in_stride[kind][1] + col * 2);
      }
      at += stride, head += stride;
      while (head >= a.heads) head -= a.heads, token++;
    }
#pragma unroll
    for (int k = 0; k < kFlight; k++) {
      if (from + k * stride >= all) break;
      const int kind = head_of[k] >= a.first[kV] ? kV : head_of[k] >= a.first[kK] ? kK : kQ;
      const int slot = min(token_of[k], kBlockTokens - 1);
      const bool normed = (a.norms >> kind) & 1, rotated = kind != kV && a.rotary > 0;
      const uint32_t raw[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
      uint32_t across[4];
      float v[8], sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        v[e] = to_float<BF16>((uint16_t)(raw[e / 2] >> (16 * (e & 1))));
        sum += v[e] * v[e];
      }
#pragma unroll
      for (int o = 1; o < LANES; o <<= 1) sum += __shfl_xor_sync(kAll, sum, o);
#pragma unroll
      for (int e = 0; e < 4; e++) across[e] = __shfl_sync(kAll, raw[e], other, LANES);
      if (!valid[k]) continue;
      uint4 y = x[k];
      if (normed || rotated) {
        const float r = normed ? rsqrtf(sum * share + a.epsilon) : 1.0f;
        const float *w = normed && kind != kV ? weight[kind] : nullptr;
        float out[8];
        if (rotated && turns) {
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const int from_col = a.interleaved ? col + (e ^ 1) : other * 8 + e;
            const int pair = a.interleaved ? pair0 + e / 2 : pair0 + e;
            const float mine = w ? v[e] * w[col + e] : v[e];
            const uint16_t h = a.interleaved ? (uint16_t)(raw[e / 2] >> (16 * ((e ^ 1) & 1)))
                                             : (uint16_t)(across[e / 2] >> (16 * (e & 1)));
            const float theirs = w ? to_float<BF16>(h) * w[from_col] : to_float<BF16>(h);
            const bool second = a.interleaved ? e & 1 : upper;
            const float s = sine[slot][pair];
            out[e] = (mine * cosine[slot][pair] + theirs * (second ? s : -s)) * r;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) out[e] = (w ? v[e] * w[col + e] : v[e]) * r;
        }
        y = make_uint4(pack2<BF16>(out[0], out[1]), pack2<BF16>(out[2], out[3]), pack2<BF16>(out[4], out[5]),
                       pack2<BF16>(out[6], out[7]));
      }
      const int own = head_of[k] - a.first[kind];
      if (a.out[kind])
        *reinterpret_cast<uint4 *>(a.out[kind] + (token0 + token_of[k]) * a.out_stride[kind][0] +
                                   own * a.out_stride[kind][1] + col * 2) = y;
      if (a.cached && kind != kQ && place_at[slot] >= 0)
        *reinterpret_cast<uint4 *>(c.memory + place_at[slot] +
                                   ((kind == kV ? c.kv_heads : 0) + own) * c.head_bytes + col * 2) = y;
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
    for (int j = 0; j < 2; j++) a.in_stride[i][j] *= 2, a.out_stride[i][j] *= 2;
    a.heads += heads;
  }
  if (a.heads == 0) return DM_OK;
  if (((uintptr_t)in->q_weight | (uintptr_t)in->k_weight) & 3)
    return fail(DM_ERR_INVALID_ARGUMENT, "norm weights must be 4-byte aligned");
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
  const int groups = kThreads / (a.dim <= 64 ? 8 : a.dim <= 128 ? 16 : 32);
  // Few tokens: their heads over several blocks, so that no thread has two; many: blocks of
  // several tokens with kFlight loads a thread at least.
  int64_t blocks = in->tokens;
  unsigned along = 1;
  a.block_tokens = 1;
  if (in->tokens * ((a.heads + groups - 1) / groups) <= 148 * 4) {
    along = (a.heads + groups - 1) / groups;
  } else {
    a.block_tokens = (int)std::min<int64_t>(kBlockTokens, std::max<int64_t>(1, in->tokens / (148 * 8)));
    blocks = (in->tokens + a.block_tokens - 1) / a.block_tokens;
  }
  const KvView view = cache ? cache->view : KvView{};
  const dim3 grid((unsigned)blocks, along);
  return in->type == DM_BF16 ? launch_rotate<true>(grid, (cudaStream_t)stream, view, a)
                             : launch_rotate<false>(grid, (cudaStream_t)stream, view, a);
}

}  // extern "C"
