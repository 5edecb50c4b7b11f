// dm_kvcache.cu -- the paged key/value cache (include/diskmule_attention.h).
//
// A call that hands out pages runs in two steps. One block plans: it checks the list, adds
// up how many fresh pages each entry needs, and ranks the free pages, so that the i-th page
// asked for is the i-th lowest free one whatever the number of threads. Many blocks then
// move rows. All of it is bound by latency (the plan: a few dependent passes over a list
// and over `references`) or by memory (the rows), and nothing waits for the host.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <new>

#include "dm_kvcache.cuh"

using dma::KvView;
using dmi::fail;

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int kSmallThreads = 128;  // on an entry of a small fork
constexpr int kFreeBatch = 8;  // pages per thread and step of the search for free ones

// Scratch of a plan, int32: header, then
//   marks  [max_sequences]   which list entry named a sequence last (to find repeats)
//   first  [max_sequences]   rank of an entry's first fresh page
//   stay   [max_sequences]   compact: leading pages that an entry keeps
//   moved  [max_sequences]   compact: blocks that have moved their rows of an entry
//   fresh  [pages]           page numbers by rank
//   owner  [pages]           list entry that a fresh page goes to
struct Plan {
  int32_t *ok, *total, *marks, *first, *stay, *moved, *fresh, *owner;
};
constexpr int kPlanHeader = 4;

size_t plan_ints(const dm_kv_cache_desc &d) {
  return kPlanHeader + 4 * (size_t)d.max_sequences + 2 * (size_t)d.pages;
}

Plan plan_of(const dm_kv_cache *c) {
  Plan p;
  p.ok = c->scratch;
  p.total = c->scratch + 1;
  p.marks = c->scratch + kPlanHeader;
  p.first = p.marks + c->desc.max_sequences;
  p.stay = p.first + c->desc.max_sequences;
  p.moved = p.stay + c->desc.max_sequences;
  p.fresh = p.moved + c->desc.max_sequences;
  p.owner = p.fresh + c->desc.pages;
  return p;
}

__device__ __forceinline__ void chain() {
  dma::let_next_start();
  dma::wait_for_previous();
}

// a + b of numbers that are not negative, at most INT32_MAX
__device__ __forceinline__ int add_upto(int a, int b) {
  return (int)min((unsigned)a + (unsigned)b, (unsigned)INT32_MAX);
}

// Inclusive sum over the block; `total` gets the block's. Every thread of the block calls it.
// A sum beyond INT32_MAX stays there (entries may ask for more pages than that together).
__device__ int block_scan(int v, int *total) {
  __shared__ int sums[kPlanThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = add_upto(v, u);
  }
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  int s = lane < kPlanThreads / 32 ? sums[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s = add_upto(s, u);
  }
  const int before = __shfl_sync(0xffffffffu, s, warp ? warp - 1 : 0);
  *total = __shfl_sync(0xffffffffu, s, 31);
  __syncthreads();
  return warp ? add_upto(v, before) : v;
}

__device__ __forceinline__ int pages_for(const KvView &c, int tokens) {
  return (tokens + c.page_tokens - 1) / c.page_tokens;
}

// `rows` rows of `vec` 16-byte vectors in each of a page's parts (layer, K or V, head): a
// thread keeps its place in a part and walks over the parts, kDepth loads in flight, so the
// loop has no division (with one: 4.7 TB/s read and written at 16 sequences of 1500 kept
// tokens, 524 KB pages; so: 6.0). Parts block, + blocks, ... of the page are this block's share,
// several at once where a part has fewer vectors than there are threads. from(r) is the source
// row's address in part 0, null for none. ONCE: nobody reads the source again.
constexpr int kDepth = 4;

template <bool ONCE>
__device__ __forceinline__ uint4 load16(const uint8_t *p) {
  const uint4 *v = reinterpret_cast<const uint4 *>(p);
  return ONCE ? __ldcs(v) : *v;
}

// `tid` of `threads` threads, as block `block` of `blocks`, take part.
template <bool ONCE, typename From>
__device__ __forceinline__ void copy_parts(const KvView &c, uint8_t *to, int rows, From from, int tid,
                                           int threads, int block, int blocks) {
  const int vec = c.head_dim / 8, chunk = rows * vec;
  const int parts = c.layers * 2 * c.kv_heads;
  const int wide = chunk < threads ? threads / chunk : 1;  // parts side by side
  const int place = wide > 1 ? tid / chunk : 0;
  if (place >= wide) return;
  const int step = blocks * wide;
  for (int in = wide > 1 ? tid % chunk : tid; in < chunk; in += threads) {
    const uint8_t *src = from(in / vec);
    if (src) {
      src += (in % vec) * 16;
      uint8_t *dst = to + (int64_t)in * 16;
      int part = block * wide + place;
      for (; part + (kDepth - 1) * step < parts; part += kDepth * step) {
        uint4 r[kDepth];
#pragma unroll
        for (int k = 0; k < kDepth; k++)
          r[k] = load16<ONCE>(src + (part + k * step) * c.head_bytes);
#pragma unroll
        for (int k = 0; k < kDepth; k++)
          *reinterpret_cast<uint4 *>(dst + (part + k * step) * c.head_bytes) = r[k];
      }
      for (; part < parts; part += step)
        *reinterpret_cast<uint4 *>(dst + part * c.head_bytes) =
            load16<ONCE>(src + part * c.head_bytes);
    }
    if (wide > 1) break;
  }
}

// Fork: the child's row, its page's references, and its part of the partial page's rows.
// `tid` of `threads` threads, as block `block` of `blocks`; the first block writes the row.
__device__ void fork_entry(const KvView &c, const Plan &p, int parent, int child, int rank, int tid,
                           int threads, int block, int blocks) {
  const int length = c.lengths[parent];
  const int full = length / c.page_tokens, rest = length % c.page_tokens;
  const int32_t *from = c.table + (int64_t)parent * c.max_pages;
  const int taken = rest ? p.fresh[rank] : -1;
  if (block == 0) {
    int32_t *to = c.table + (int64_t)child * c.max_pages;
    for (int j = tid; j < c.max_pages; j += threads) {
      int page = -1;
      if (j < full) {
        page = from[j];
        if ((unsigned)page < (unsigned)c.pages) atomicAdd(c.references + page, 1);
      } else if (j == full && rest) {
        page = taken;
        c.references[page] = 1;
      }
      to[j] = page;
    }
    if (tid == 0) c.lengths[child] = length;
  }
  if (!rest) return;
  const int old = from[full];
  if ((unsigned)old >= (unsigned)c.pages) return;
  const uint8_t *src = c.memory + old * c.page_bytes;
  const int64_t row_bytes = c.head_dim * 2;
  copy_parts<false>(c, c.memory + taken * c.page_bytes, rest, [&](int r) { return src + r * row_bytes; },
                    tid, threads, block, blocks);
}

// block (x, i) takes its part of entry i
__global__ void __launch_bounds__(kCopyThreads)
fork_kernel(KvView c, Plan p, const int32_t *parents, const int32_t *children) {
  chain();
  if (!*p.ok) return;
  const int i = blockIdx.y;
  fork_entry(c, p, parents[i], children[i], p.first[i], threadIdx.x, kCopyThreads, blockIdx.x, gridDim.x);
}

enum PlanOp { kFork, kForkSmall, kExtend, kCompact };  // kForkSmall copies here, too

struct PlanArgs {
  const int32_t *rows;     // children, or the sequences
  const int32_t *other;    // fork: parents; extend: counts; compact: keep_offsets
  const int32_t *keep;     // compact
  int64_t kept;
  int32_t n;
};

// Compact: keep[0..count) ascends, so keep[j] == j holds for a leading part and fails
// behind it. The warp looks for the end of that part, 32 probes at a time.
__device__ int leading_same(const int32_t *keep, int count) {
  const int lane = threadIdx.x & 31;
  int low = 0, high = count;  // all of [0, low) are the same, high is not (or is the end)
  while (low < high) {
    const int step = (high - low + 31) / 32;
    const int at = low + step * (lane + 1) - 1;
    const bool same = at < high && keep[at] == at;
    const int run = __popc(__ballot_sync(0xffffffffu, same));  // the first `run` probes hold
    const int next = low + run * step;
    high = min(high, low + step * (run + 1) - 1);
    low = next;
  }
  return low;
}

// Whether keep[j] opens an entry's list; offsets that do not ascend give any answer.
__device__ bool opens_entry(const int32_t *offsets, int n, int64_t j) {
  int low = 0, high = n;  // offsets[low] <= j
  while (low < high) {
    const int mid = (low + high + 1) >> 1;
    if (offsets[mid] <= j) low = mid;
    else high = mid - 1;
  }
  return offsets[low] == j;
}

// One block. ok = 1 and the plan where the whole call can be done, else 0 and a status bit.
// Extend has no rows to move and is done here.
template <int OP>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(KvView c, Plan p, PlanArgs a) {
  __shared__ int bad;
  const int tid = threadIdx.x;
  chain();
  // the first pages' references come in beside the list (most calls need no others)
  int refs[kFreeBatch];
#pragma unroll
  for (int k = 0; k < kFreeBatch; k++)
    refs[k] = tid * kFreeBatch + k < c.pages ? c.references[tid * kFreeBatch + k] : 1;
  if (tid == 0) bad = 0;
  __syncthreads();
  for (int i = tid; i < a.n; i += kPlanThreads) {
    const int row = a.rows[i];
    if (row < 0 || row >= c.max_sequences) atomicOr(&bad, DM_KV_BAD_SEQUENCE);
    else p.marks[row] = i;
  }
  __syncthreads();
  const bool listed = !bad;
  __syncthreads();
  int total = 0;
  if (listed) {
    if (OP == kCompact) {  // one warp per sequence
      for (int i = tid >> 5; i < a.n; i += kPlanThreads / 32) {
        const int row = a.rows[i];
        const int k0 = a.other[i], count = a.other[i + 1] - k0;
        if (k0 < 0 || count < 0 || (int64_t)k0 + count > a.kept || count > c.lengths[row] ||
            c.lengths[row] > c.max_pages * (int64_t)c.page_tokens) {
          if ((tid & 31) == 0) atomicOr(&bad, DM_KV_BAD_TOKEN);
          continue;
        }
        // the ends of the list come in beside the search, which reads nothing outside it
        const int head = count ? a.keep[k0] : 0, tail = count ? a.keep[k0 + count - 1] : -1;
        const int same = leading_same(a.keep + k0, count);
        if ((tid & 31) == 0 && (head < 0 || tail >= c.lengths[row])) atomicOr(&bad, DM_KV_BAD_TOKEN);
        int stay = same / c.page_tokens;
        if (same == count) {  // only the tail goes
          stay = pages_for(c, count);
          // a partial last page that others still hold is copied
          if (count % c.page_tokens) {
            const int last = c.table[(int64_t)row * c.max_pages + stay - 1];
            if ((unsigned)last < (unsigned)c.pages && c.references[last] > 1) stay--;
          }
        }
        if ((tid & 31) == 0) p.stay[i] = stay, p.moved[i] = 0;
      }
      // Between its first and last token, which are in range, an entry's list ascends. All
      // lists in one pass, kSteps loads of a thread in flight: a step down is rare where no new
      // entry begins.
      constexpr int kSteps = 8;
      const int64_t end = min((int64_t)a.other[a.n], a.kept) - 1;
      for (int64_t j0 = (int64_t)max(a.other[0], 0) + tid; j0 < end; j0 += kSteps * kPlanThreads) {
        unsigned down = 0;
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
          const int64_t j = j0 + k * kPlanThreads;
          if (j < end && a.keep[j] >= a.keep[j + 1]) down |= 1u << k;
        }
        for (; down; down &= down - 1)
          if (!opens_entry(a.other, a.n, j0 + (__ffs(down) - 1) * kPlanThreads + 1)) atomicOr(&bad, DM_KV_BAD_TOKEN);
      }
      __syncthreads();
    }
    for (int i0 = 0; i0 < a.n; i0 += kPlanThreads) {
      const int i = i0 + tid;
      int need = 0;
      if (i < a.n && !(OP == kCompact && bad)) {
        const int row = a.rows[i];
        int wrong = p.marks[row] == i ? 0 : DM_KV_BAD_SEQUENCE;
        if (OP == kFork || OP == kForkSmall) {
          // a parent is no target of this call
          const int parent = a.other[i];
          bool fit = parent >= 0 && parent < c.max_sequences && c.lengths[row] == 0;
          if (fit) {
            const int m = p.marks[parent], length = c.lengths[parent];
            fit = !(m >= 0 && m < a.n && a.rows[m] == parent) && length >= 0 &&
                  length <= c.max_pages * (int64_t)c.page_tokens;
            need = fit && length % c.page_tokens != 0;
          }
          if (!fit) wrong |= DM_KV_BAD_SEQUENCE;
        } else if (OP == kExtend) {
          const int old = c.lengths[row], count = a.other[i];
          if (old < 0 || count < 0 || count > c.max_pages * (int64_t)c.page_tokens - old)
            wrong |= count < 0 ? DM_KV_BAD_TOKEN : DM_KV_TOO_LONG;
          else
            need = pages_for(c, old + count) - pages_for(c, old);
        } else {
          need = pages_for(c, a.other[i + 1] - a.other[i]) - p.stay[i];
        }
        if (wrong) atomicOr(&bad, wrong);
      }
      int sum;
      const int upto = block_scan(need, &sum), before = total;
      total = add_upto(total, sum);
      if (total > c.pages) break;
      if (i < a.n) p.first[i] = before + upto - need;
      for (int r = 0; r < need; r++) p.owner[before + upto - need + r] = i;
    }
  }
  __syncthreads();
  // rank the free pages until there are enough
  int found = 0;
  if (!bad && total <= c.pages) {
    for (int p0 = 0; p0 < c.pages && found < total; p0 += kPlanThreads * kFreeBatch) {
      int mine = 0;
      const int at = p0 + tid * kFreeBatch;
      if (p0 > 0)
#pragma unroll
        for (int k = 0; k < kFreeBatch; k++) refs[k] = at + k < c.pages ? c.references[at + k] : 1;
#pragma unroll
      for (int k = 0; k < kFreeBatch; k++) mine += refs[k] == 0;
      int sum;
      int rank = found + block_scan(mine, &sum) - mine;
#pragma unroll
      for (int k = 0; k < kFreeBatch; k++)
        if (refs[k] == 0) {
          if (rank < total) p.fresh[rank] = at + k;
          rank++;
        }
      found += sum;
    }
  }
  __syncthreads();
  const bool ok = !bad && found >= total;
  if (tid == 0) {
    *p.ok = ok;
    *p.total = ok ? total : 0;
    if (bad) atomicOr(c.status, bad);
    else if (!ok) atomicOr(c.status, DM_KV_OUT_OF_PAGES);
  }
  if (OP == kForkSmall && ok) {
    __syncthreads();  // children are empty and no parents: in any order
    for (int i = tid / kSmallThreads; i < a.n; i += kPlanThreads / kSmallThreads)
      fork_entry(c, p, a.other[i], a.rows[i], p.first[i], tid % kSmallThreads, kSmallThreads, 0, 1);
  }
  if (OP == kExtend && ok) {
    for (int f = tid; f < total; f += kPlanThreads) {
      const int i = p.owner[f], row = a.rows[i], page = p.fresh[f];
      c.table[(int64_t)row * c.max_pages + pages_for(c, c.lengths[row]) + f - p.first[i]] = page;
      c.references[page] = 1;
    }
    __syncthreads();
    for (int i = tid; i < a.n; i += kPlanThreads) c.lengths[a.rows[i]] += a.other[i];
  }
}

// Compact, once the rows of entry i have moved: let go of the old pages and write the row.
__device__ void settle_entry(const KvView &c, const Plan &p, const PlanArgs &a, int i) {
  const int row = a.rows[i], count = a.other[i + 1] - a.other[i];
  const int stay = p.stay[i], now = pages_for(c, count), before = pages_for(c, c.lengths[row]);
  int32_t *entries = c.table + (int64_t)row * c.max_pages;
  for (int j = stay + threadIdx.x; j < c.max_pages; j += blockDim.x) {
    const int old = entries[j];
    if (j < before && (unsigned)old < (unsigned)c.pages) atomicSub(c.references + old, 1);
    int page = -1;
    if (j < now) {
      page = p.fresh[p.first[i] + j - stay];
      c.references[page] = 1;
    }
    entries[j] = page;
  }
  __syncthreads();
  if (threadIdx.x == 0) c.lengths[row] = count;
}

// Compact: jobs (along y) are the plan's fresh pages, then the entries without one. Block
// (x, f) gathers its part of page f; the last block of an entry's pages settles it.
__global__ void __launch_bounds__(kCopyThreads)
gather_kernel(KvView c, Plan p, PlanArgs a) {
  chain();
  if (!*p.ok) return;
  const int total = *p.total;
  __shared__ int64_t source[256];  // of each row of the page, -1 where it has none
  __shared__ int last;
  for (int f = blockIdx.y; f < total + a.n; f += gridDim.y) {
    if (f >= total) {
      const int i = f - total;
      if (blockIdx.x == 0 && pages_for(c, a.other[i + 1] - a.other[i]) == p.stay[i]) settle_entry(c, p, a, i);
      continue;
    }
    const int i = p.owner[f], row = a.rows[i];
    const int k0 = a.other[i], count = a.other[i + 1] - k0;
    const int j0 = (p.stay[i] + f - p.first[i]) * c.page_tokens;
    const int used = min(c.page_tokens, count - j0);
    for (int r = threadIdx.x; r < used; r += kCopyThreads) {
      const int token = a.keep[k0 + j0 + r];
      const int page = c.table[(int64_t)row * c.max_pages + token / c.page_tokens];
      source[r] = (unsigned)page < (unsigned)c.pages
                      ? page * c.page_bytes + (int64_t)(token % c.page_tokens) * c.head_dim * 2 : -1;
    }
    __syncthreads();
    uint8_t *dst = c.memory + p.fresh[f] * c.page_bytes;
    copy_parts<true>(c, dst, used, [&](int r) -> const uint8_t * {
      return source[r] < 0 ? nullptr : c.memory + source[r];
    }, threadIdx.x, kCopyThreads, blockIdx.x, gridDim.x);
    // everything that this block reads of the entry has been read
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
      const int pages = pages_for(c, count) - p.stay[i];
      last = atomicAdd(p.moved + i, 1) == pages * (int)gridDim.x - 1;
    }
    __syncthreads();
    if (last) settle_entry(c, p, a, i);
    __syncthreads();
  }
}

// Free: block i takes the length of its sequence (a repeat finds zero) and lets go.
__global__ void __launch_bounds__(kCopyThreads) free_kernel(KvView c, const int32_t *rows) {
  __shared__ int held;
  chain();
  const int row = rows[blockIdx.x];
  if (row < 0 || row >= c.max_sequences) {
    if (threadIdx.x == 0) atomicOr(c.status, DM_KV_BAD_SEQUENCE);
    return;
  }
  if (threadIdx.x == 0) held = min(pages_for(c, atomicExch(c.lengths + row, 0)), c.max_pages);
  __syncthreads();
  int32_t *entries = c.table + (int64_t)row * c.max_pages;
  for (int j = threadIdx.x; j < held; j += blockDim.x) {
    const int page = entries[j];
    if ((unsigned)page < (unsigned)c.pages) atomicSub(c.references + page, 1);
    entries[j] = -1;
  }
}

struct WriteArgs {
  const uint8_t *k, *v;
  int64_t stride[2][2];  // [K, V][token, head], elements
  const int32_t *rows, *offsets;
  int32_t n, layer;
  int64_t tokens;
};

// Write: one thread per 16-byte vector of a token's keys and values.
__global__ void __launch_bounds__(kCopyThreads) write_kernel(KvView c, WriteArgs a) {
  chain();
  const int vec = c.head_dim / 8, half = c.kv_heads * vec;
  const int64_t at = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x;
  const int64_t t = at / (2 * half);
  if (t >= a.tokens) return;
  const int i = (int)(at - t * 2 * half);
  // the sequence whose rows hold t: the last offset that is not above it
  int low = 0, high = a.n;
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (a.offsets[mid] <= t) low = mid;
    else high = mid;
  }
  const int row = a.rows[low], o0 = a.offsets[low], o1 = a.offsets[low + 1];
  int64_t place = -1;
  int page = -1;
  if (row >= 0 && row < c.max_sequences && t >= o0 && t < o1) {
    const int length = c.lengths[row];
    place = length - ((int64_t)o1 - t);
    if (place >= 0 && place < length && place / c.page_tokens < c.max_pages)
      page = c.table[(int64_t)row * c.max_pages + place / c.page_tokens];
  }
  if ((unsigned)page >= (unsigned)c.pages) {
    if (i == 0) atomicOr(c.status, DM_KV_BAD_TOKEN);
    return;
  }
  const int which = i >= half, head = (i - which * half) / vec, in = (i - which * half) % vec;
  const uint8_t *src = (which ? a.v : a.k) +
                       (t * a.stride[which][0] + head * a.stride[which][1]) * 2 + in * 16;
  uint8_t *dst = c.memory + page * c.page_bytes + a.layer * c.layer_bytes +
                 (which * c.kv_heads + head) * c.head_bytes +
                 (place % c.page_tokens) * c.head_dim * 2 + in * 16;
  *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(src);
}

__global__ void __launch_bounds__(kCopyThreads)
copy_pages_kernel(KvView c, const int32_t *source, const int32_t *target) {
  chain();
  const int from = source[blockIdx.y], to = target[blockIdx.y];
  if ((unsigned)from >= (unsigned)c.pages || (unsigned)to >= (unsigned)c.pages) {
    if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(c.status, DM_KV_BAD_TOKEN);
    return;
  }
  const uint4 *src = reinterpret_cast<const uint4 *>(c.memory + from * c.page_bytes);
  uint4 *dst = reinterpret_cast<uint4 *>(c.memory + to * c.page_bytes);
  const int64_t total = c.page_bytes / 16, stride = (int64_t)gridDim.x * kCopyThreads;
  for (int64_t v0 = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; v0 < total; v0 += 4 * stride) {
    uint4 r[4];
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (v0 + k * stride < total) r[k] = src[v0 + k * stride];
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (v0 + k * stride < total) dst[v0 + k * stride] = r[k];
  }
}

// Blocks per page or row so that about `blocks` run in all, each with at least 4 vectors per
// thread.
int blocks_along(int64_t vectors, int64_t items, int64_t blocks) {
  const int64_t fit = std::max<int64_t>(1, vectors / (4 * kCopyThreads));
  return (int)std::max<int64_t>(1, std::min(fit, blocks / std::max<int64_t>(1, items)));
}
constexpr int kGridBlocks = 148 * 8;
constexpr int kSmallForks = 16;
constexpr int64_t kSmallCopy = 512 * 1024, kSmallRows = 16384;  // bytes of pages, table entries

template <typename... Params, typename... Args>
int32_t launch(void (*kernel)(Params...), dim3 grid, int threads, void *stream, const Args &...args) {
  return dma::launch_chained("cache launch", kernel, grid, threads, 0, (cudaStream_t)stream, args...);
}

int32_t check_list(const dm_kv_cache *cache, const void *list, int32_t n) {
  if (!cache) return fail(DM_ERR_INVALID_ARGUMENT, "null cache");
  if (n < 0) return fail(DM_ERR_ELEMENT_COUNT, "a list of %d sequences", n);
  if (n > 0 && !list) return fail(DM_ERR_INVALID_ARGUMENT, "null list");
  if (n > cache->desc.max_sequences)
    return fail(DM_ERR_ELEMENT_COUNT, "%d sequences, and the cache has %d", n,
                cache->desc.max_sequences);
  return DM_OK;
}

template <typename T>
int32_t provide(void *given, T **slot, bool *own, size_t count, int fill, cudaStream_t stream) {
  *slot = (T *)given;
  if (given) return DM_OK;
  void *p = nullptr;
  if (cudaMalloc(&p, count * sizeof(T)) != cudaSuccess) {
    cudaGetLastError();
    return fail(DM_ERR_ALLOCATION, "could not allocate %zu bytes for the cache", count * sizeof(T));
  }
  *slot = (T *)p;
  *own = true;
  DM_CUDA(cudaMemsetAsync(p, fill, count * sizeof(T), stream), "cache set-up");
  return DM_OK;
}

}  // namespace

extern "C" {

int32_t dm_kv_cache_create(dm_cuda_context *ctx, const dm_kv_cache_desc *d, dm_kv_cache **out) {
  if (!ctx || !d || !out) return fail(DM_ERR_INVALID_ARGUMENT, "null argument");
  *out = nullptr;
  if (d->type != DM_BF16 && d->type != DM_F16)
    return fail(DM_ERR_UNSUPPORTED_TENSOR_TYPE, "a cache holds bf16 or f16");
  if (d->layers <= 0 || d->kv_heads <= 0 || d->pages <= 0 || d->max_sequences <= 0 || d->max_pages <= 0)
    return fail(DM_ERR_EMPTY_INPUT, "an empty cache");
  if (d->head_dim <= 0 || d->head_dim % 8 || d->head_dim > 256)
    return fail(DM_ERR_ELEMENT_COUNT, "head_dim %d is not a multiple of 8 up to 256", d->head_dim);
  if (d->page_tokens < 16 || d->page_tokens > 256 || (d->page_tokens & (d->page_tokens - 1)))
    return fail(DM_ERR_ELEMENT_COUNT, "page_tokens %d is not a power of two from 16 to 256",
                d->page_tokens);
  const int64_t head_bytes = (int64_t)d->page_tokens * d->head_dim * 2;
  const int64_t layer_bytes = head_bytes * 2 * d->kv_heads;
  // pages, rows of a page and a table row's tokens are counted in 32 bits
  if (d->pages > 1 << 30) return fail(DM_ERR_OVERFLOW, "more than 2^30 pages");
  if (layer_bytes > ((int64_t)1 << 32) / d->layers || (int64_t)d->layers * 2 * d->kv_heads > INT32_MAX)
    return fail(DM_ERR_OVERFLOW, "a page of more than 4 GB");
  if ((int64_t)d->max_pages * d->page_tokens > dma::kMostTokens)
    return fail(DM_ERR_OVERFLOW, "a sequence of more than %d tokens", dma::kMostTokens);
  if ((uintptr_t)d->memory & 15)
    return fail(DM_ERR_INVALID_ARGUMENT, "cache memory must be 16-byte aligned");
  dm_kv_cache *c = new (std::nothrow) dm_kv_cache;
  if (!c) return fail(DM_ERR_ALLOCATION, "could not allocate a cache");
  c->desc = *d;
  c->ctx = ctx;
  dmi::retain_context(ctx);
  cudaSetDevice(ctx->device);
  const size_t page_bytes = (size_t)(layer_bytes * d->layers);
  uint8_t *memory = nullptr;
  bool own_scratch = false;
  int32_t rc = provide(d->memory, &memory, &c->own_memory, page_bytes * d->pages, 0, ctx->stream);
  c->desc.memory = memory;
  if (!rc)
    rc = provide(d->page_table, &c->desc.page_table, &c->own_table,
                 (size_t)d->max_sequences * d->max_pages, 0xff, ctx->stream);
  if (!rc)
    rc = provide(d->lengths, &c->desc.lengths, &c->own_lengths, (size_t)d->max_sequences, 0,
                 ctx->stream);
  if (!rc)
    rc = provide(d->references, &c->desc.references, &c->own_references, (size_t)d->pages, 0,
                 ctx->stream);
  // the plan and, behind it, the status word
  if (!rc) rc = provide(nullptr, &c->scratch, &own_scratch, plan_ints(*d) + 1, 0, ctx->stream);
  if (!rc && cudaStreamSynchronize(ctx->stream) != cudaSuccess)
    rc = dmi::cuda_fail(cudaGetLastError(), "cache set-up");
  if (rc) {
    dm_kv_cache_destroy(c);
    return rc;
  }
  KvView &v = c->view;
  v.memory = memory;
  v.table = c->desc.page_table;
  v.lengths = c->desc.lengths;
  v.references = c->desc.references;
  v.status = c->scratch + plan_ints(*d);
  v.layers = d->layers;
  v.kv_heads = d->kv_heads;
  v.head_dim = d->head_dim;
  v.page_tokens = d->page_tokens;
  v.pages = d->pages;
  v.max_sequences = d->max_sequences;
  v.max_pages = d->max_pages;
  v.head_bytes = head_bytes;
  v.layer_bytes = layer_bytes;
  v.page_bytes = (int64_t)page_bytes;
  *out = c;
  return DM_OK;
}

void dm_kv_cache_destroy(dm_kv_cache *c) {
  if (!c) return;
  cudaSetDevice(c->ctx->device);
  if (c->own_memory) cudaFree(c->desc.memory);
  if (c->own_table) cudaFree(c->desc.page_table);
  if (c->own_lengths) cudaFree(c->desc.lengths);
  if (c->own_references) cudaFree(c->desc.references);
  if (c->scratch) cudaFree(c->scratch);
  dmi::release_context(c->ctx);
  delete c;
}

int32_t dm_kv_cache_describe(const dm_kv_cache *c, dm_kv_cache_desc *desc) {
  if (!c || !desc) return fail(DM_ERR_INVALID_ARGUMENT, "null argument");
  *desc = c->desc;
  return DM_OK;
}

int32_t dm_kv_cache_status(dm_kv_cache *c, int32_t *bits, void *stream) {
  if (!c || !bits) return fail(DM_ERR_INVALID_ARGUMENT, "null argument");
  cudaSetDevice(c->ctx->device);
  cudaStream_t s = (cudaStream_t)stream;
  DM_CUDA(cudaMemcpyAsync(bits, c->view.status, 4, cudaMemcpyDeviceToHost, s), "cache status");
  DM_CUDA(cudaMemsetAsync(c->view.status, 0, 4, s), "cache status");
  DM_CUDA(cudaStreamSynchronize(s), "cache status");
  return DM_OK;
}

int32_t dm_kv_cache_extend(dm_kv_cache *c, const int32_t *sequences, const int32_t *counts,
                           int32_t n, void *stream) {
  if (int32_t rc = check_list(c, sequences, n)) return rc;
  if (n == 0) return DM_OK;
  if (!counts) return fail(DM_ERR_INVALID_ARGUMENT, "null counts");
  cudaSetDevice(c->ctx->device);
  return launch(plan_kernel<kExtend>, 1, kPlanThreads, stream, c->view, plan_of(c),
                PlanArgs{sequences, counts, nullptr, 0, n});
}

int32_t dm_kv_cache_write(dm_kv_cache *c, int32_t layer, const void *k, const void *v,
                          const int64_t *k_stride, const int64_t *v_stride,
                          const int32_t *sequences, const int32_t *offsets, int32_t n,
                          int64_t tokens, void *stream) {
  if (int32_t rc = check_list(c, sequences, n)) return rc;
  if (layer < 0 || layer >= c->desc.layers)
    return fail(DM_ERR_INVALID_LAYER, "layer %d of %d", layer, c->desc.layers);
  if (tokens < 0 || tokens > INT32_MAX) return fail(DM_ERR_ELEMENT_COUNT, "a bad number of tokens");
  if (n == 0 || tokens == 0) return DM_OK;
  if (!k || !v || !offsets) return fail(DM_ERR_INVALID_ARGUMENT, "null argument");
  WriteArgs a{(const uint8_t *)k, (const uint8_t *)v, {}, sequences, offsets, n, layer, tokens};
  const int64_t *given[2] = {k_stride, v_stride};
  for (int i = 0; i < 2; i++) {
    a.stride[i][0] = given[i] && (given[i][0] || given[i][1])
                         ? given[i][0] : (int64_t)c->desc.kv_heads * c->desc.head_dim;
    a.stride[i][1] = given[i] && (given[i][0] || given[i][1]) ? given[i][1] : c->desc.head_dim;
    if (a.stride[i][0] % 8 || a.stride[i][1] % 8)
      return fail(DM_ERR_INVALID_ARGUMENT, "strides must be multiples of 8 elements");
  }
  if (((uintptr_t)k | (uintptr_t)v) & 15)
    return fail(DM_ERR_INVALID_ARGUMENT, "keys and values must be 16-byte aligned");
  cudaSetDevice(c->ctx->device);
  const int64_t vectors = tokens * c->desc.kv_heads * c->desc.head_dim / 4;  // K and V
  const int64_t blocks = (vectors + kCopyThreads - 1) / kCopyThreads;
  if (blocks > INT32_MAX) return fail(DM_ERR_OVERFLOW, "too many tokens in one write");
  return launch(write_kernel, (unsigned)blocks, kCopyThreads, stream, c->view, a);
}

int32_t dm_kv_cache_fork(dm_kv_cache *c, const int32_t *parents, const int32_t *children,
                         int32_t n, void *stream) {
  if (int32_t rc = check_list(c, children, n)) return rc;
  if (n == 0) return DM_OK;
  if (!parents) return fail(DM_ERR_INVALID_ARGUMENT, "null parents");
  if (n > 65535) return fail(DM_ERR_ELEMENT_COUNT, "%d forks in one call", n);
  cudaSetDevice(c->ctx->device);
  const PlanArgs a{children, parents, nullptr, 0, n};
  // A few small forks are done by the plan's block: a launch less, where the caller's side bounds
  // a call (free and fork of 8 entries with 32 KB pages 10.8 us instead of 13.4). On the GPU it
  // gains nothing and loses by size. Free and fork there, us, and with a kernel for the rows: 8
  // entries with 32 KB pages 9.5 (9.4), with table rows of 2048 entries 10.3 (9.7), of 16384
  // 17.4 (12.0); 16 entries with 4 KB pages 9.9 (9.4), 64 of them 19.2 (9.8); 2 with 256 KB pages
  // 10.6 (9.6).
  if (n <= kSmallForks && n * c->view.page_bytes <= kSmallCopy && (int64_t)n * c->desc.max_pages <= kSmallRows)
    return launch(plan_kernel<kForkSmall>, 1, kPlanThreads, stream, c->view, plan_of(c), a);
  if (int32_t rc = launch(plan_kernel<kFork>, 1, kPlanThreads, stream, c->view, plan_of(c), a)) return rc;
  // half a page is copied on average
  const dim3 grid(blocks_along(c->view.page_bytes / 32, n, kGridBlocks), n);
  return launch(fork_kernel, grid, kCopyThreads, stream, c->view, plan_of(c), parents, children);
}

int32_t dm_kv_cache_compact(dm_kv_cache *c, const int32_t *sequences, const int32_t *keep_offsets,
                            const int32_t *keep, int32_t n, int64_t kept, void *stream) {
  if (int32_t rc = check_list(c, sequences, n)) return rc;
  if (kept < 0 || kept > INT32_MAX) return fail(DM_ERR_ELEMENT_COUNT, "a bad number of kept tokens");
  if (n == 0) return DM_OK;
  if (!keep_offsets || (kept && !keep)) return fail(DM_ERR_INVALID_ARGUMENT, "null keep list");
  cudaSetDevice(c->ctx->device);
  const PlanArgs a{sequences, keep_offsets, keep, kept, n};
  if (int32_t rc = launch(plan_kernel<kCompact>, 1, kPlanThreads, stream, c->view, plan_of(c), a))
    return rc;
  // at most this many fresh pages
  const int64_t fresh = std::min<int64_t>(c->desc.pages, kept / c->desc.page_tokens + n);
  const dim3 grid(blocks_along(c->view.page_bytes / 16, fresh, kGridBlocks),
                  (unsigned)std::min<int64_t>(fresh + n, 65535));
  return launch(gather_kernel, grid, kCopyThreads, stream, c->view, plan_of(c), a);
}

int32_t dm_kv_cache_free(dm_kv_cache *c, const int32_t *sequences, int32_t n, void *stream) {
  if (int32_t rc = check_list(c, sequences, n)) return rc;
  if (n == 0) return DM_OK;
  cudaSetDevice(c->ctx->device);
  return launch(free_kernel, n, kCopyThreads, stream, c->view, sequences);
}

int32_t dm_kv_cache_copy_pages(dm_kv_cache *c, const int32_t *source, const int32_t *target,
                               int32_t n, void *stream) {
  if (!c) return fail(DM_ERR_INVALID_ARGUMENT, "null cache");
  if (n < 0 || n > c->desc.pages || n > 65535)
    return fail(DM_ERR_ELEMENT_COUNT, "a list of %d pages", n);
  if (n == 0) return DM_OK;
  if (!source || !target) return fail(DM_ERR_INVALID_ARGUMENT, "null list");
  cudaSetDevice(c->ctx->device);
  const dim3 grid(blocks_along(c->view.page_bytes / 16, n, kGridBlocks), n);
  return launch(copy_pages_kernel, grid, kCopyThreads, stream, c->view, source, target);
}

}  // extern "C"
