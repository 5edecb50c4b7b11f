/*
 * diskmule_attention.h -- attention and its key/value cache on the device: the half of a
 * decode stack that comes before the routed feed-forward block (diskmule_cuda.h).
 *
 *   dm_attention_prompt   attention over whole prompts: packed sequences of different
 *                         lengths, grouped heads, causal and sliding-window masks
 *   dm_kv_cache_*         a paged cache: extend, write, fork, compact, free, copy pages
 *   dm_attention_decode   one query token per sequence against the cache; tokens that all
 *                         sequences share are read once for the whole batch
 *
 * Conventions:
 *   - tensors are DM_BF16 or DM_F16, the same type on input and output; scores, softmax
 *     statistics and output sums are f32;
 *   - query head h reads key/value head h / (heads / kv_heads);
 *   - lse (optional) is the natural logarithm of a row's sum of exp(score), f32; a row that
 *     sees no key gets zeros and -infinity;
 *   - a sequence, and a packed tensor, has at most 2^31 - 4097 tokens;
 *   - what a mask hides has no influence, whatever it holds (NaN and infinities included);
 *   - calls are stream-ordered, allocate nothing and may be captured into a CUDA graph;
 *   - arguments are checked before any launch; what only the device can see is range-checked
 *     there. Cache calls and decode report lists, positions and pages out of range through
 *     the cache's status word (dm_kv_cache_status); prompt offsets are limited to the tensors.
 */
#ifndef DISKMULE_ATTENTION_H
#define DISKMULE_ATTENTION_H

#include <stdint.h>

#include "diskmule_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct dm_kv_cache dm_kv_cache;

/* ---- prompts ---------------------------------------------------------------------- */

/* q [q_tokens, heads, head_dim], k and v [k_tokens, kv_heads, head_dim], out like q, lse
 * [q_tokens, heads]. Strides are in elements, {token, head}; {0, 0} means contiguous.
 * Pointers are 16-byte aligned and strides multiples of 8 elements; head_dim is a multiple
 * of 8 up to 256; at most 128 query heads per key/value head and 2^20 sequences.
 * Sequence s owns query rows [q_offsets[s], q_offsets[s + 1]) and key rows
 * [k_offsets[s], k_offsets[s + 1]) (device int32, [sequences + 1], ascending from >= 0;
 * k_offsets NULL = q_offsets). The last query row is aligned with the last key: query row
 * i of Lq stands at position p = i + Lk - Lq and, if causal, sees keys j <= p; window > 0
 * also hides keys j <= p - window. scale multiplies the scores (0 = 1 / sqrt(head_dim)). */
typedef struct {
  int32_t type, heads, kv_heads, head_dim;
  int32_t sequences, causal, window;
  float scale;
  int64_t q_tokens, k_tokens;
  const void *q, *k, *v;
  void *out;
  float *lse;
  int64_t q_stride[2], k_stride[2], v_stride[2], out_stride[2];
  const int32_t *q_offsets, *k_offsets;
} dm_attention_prompt_desc;

DM_API int32_t dm_attention_prompt(dm_cuda_context *ctx, const dm_attention_prompt_desc *desc,
                                   void *stream);
/* Waits for `stream`; DM_ERR_TIMEOUT if a bounded wait inside an attention kernel of this
 * context has run out since the last call (its output is then undefined). */
DM_API int32_t dm_attention_status(dm_cuda_context *ctx, void *stream);

/* ---- the paged cache ---------------------------------------------------------------- */

/* memory      [pages][layers][2 (K, V)][kv_heads][page_tokens][head_dim] of `type`
 * page_table  [max_sequences][max_pages] int32: the pages of each sequence, -1 behind them
 * lengths     [max_sequences] int32 tokens
 * references  [pages] int32: sequences that hold the page; 0 = free
 * All four are device pointers. Any that is NULL at dm_kv_cache_create is allocated (an
 * empty table, lengths and references of zero) and freed with the cache; given ones stay the
 * caller's and are taken as they are. page_tokens is a power of two from 16 to 256.
 *
 * The calls below take device int32 lists and update the tables on the device. Pages are
 * handed out in list order, the lowest free page first. Extend, fork and compact change
 * nothing and set a bit of the status word where they need more pages than are free, or where
 * a list holds a bad or repeated sequence, a bad count or a token out of range or order.
 * Free, write and copy_pages do what can be done and set the bit for the rest; a sequence that
 * is named twice is freed once. Fork and copy_pages take at most 65535 entries. Calls on one
 * cache are ordered by the caller (one stream, or events). A last page that is only partly
 * filled belongs to one sequence alone. */
typedef struct {
  int32_t type, layers, kv_heads, head_dim, page_tokens, pages, max_sequences, max_pages;
  void *memory;
  int32_t *page_table, *lengths, *references;
} dm_kv_cache_desc;

enum {
  DM_KV_OUT_OF_PAGES = 1,  /* not enough free pages */
  DM_KV_BAD_SEQUENCE = 2,  /* out of range, named twice, or a fork target that is not empty */
  DM_KV_TOO_LONG = 4,      /* a sequence would outgrow its row of the page table */
  DM_KV_BAD_TOKEN = 8,     /* a token position, count, offset or page out of range or order */
};

DM_API int32_t dm_kv_cache_create(dm_cuda_context *ctx, const dm_kv_cache_desc *desc,
                                  dm_kv_cache **out);
DM_API void dm_kv_cache_destroy(dm_kv_cache *cache);
/* The geometry and the four device pointers. */
DM_API int32_t dm_kv_cache_describe(const dm_kv_cache *cache, dm_kv_cache_desc *desc);
/* Waits for `stream`, returns the DM_KV_* bits in *bits and clears them. */
DM_API int32_t dm_kv_cache_status(dm_kv_cache *cache, int32_t *bits, void *stream);

/* lengths[sequences[i]] += counts[i]; pages for the new tokens (their content is not
 * written). */
DM_API int32_t dm_kv_cache_extend(dm_kv_cache *cache, const int32_t *sequences,
                                  const int32_t *counts, int32_t n, void *stream);
/* Keys and values of one layer for the LAST offsets[i + 1] - offsets[i] tokens of
 * sequences[i]: rows offsets[i] .. of k and v [tokens, kv_heads, head_dim] (strides as above,
 * k_stride / v_stride NULL = contiguous); tokens is the number of rows, offsets[n]. */
DM_API int32_t dm_kv_cache_write(dm_kv_cache *cache, int32_t layer, const void *k, const void *v,
                                 const int64_t *k_stride, const int64_t *v_stride,
                                 const int32_t *sequences, const int32_t *offsets, int32_t n,
                                 int64_t tokens, void *stream);
/* children[i] (empty) becomes a copy of parents[i]: full pages are shared, the used rows of a
 * partial last page are copied to a fresh page. */
DM_API int32_t dm_kv_cache_fork(dm_kv_cache *cache, const int32_t *parents,
                                const int32_t *children, int32_t n, void *stream);
/* sequences[i] keeps the tokens keep[keep_offsets[i]] < ... < keep[keep_offsets[i + 1] - 1]
 * of its present ones, in that order. Leading pages whose tokens all stay in place are kept;
 * the others are gathered into fresh pages and let go. kept is the length of keep,
 * keep_offsets[n]. */
DM_API int32_t dm_kv_cache_compact(dm_kv_cache *cache, const int32_t *sequences,
                                   const int32_t *keep_offsets, const int32_t *keep, int32_t n,
                                   int64_t kept, void *stream);
/* Empties the sequences; pages that no other sequence holds become free. */
DM_API int32_t dm_kv_cache_free(dm_kv_cache *cache, const int32_t *sequences, int32_t n,
                                void *stream);
/* Page target[i] = page source[i], all layers. No page is both source and target, and no
 * target is named twice. */
DM_API int32_t dm_kv_cache_copy_pages(dm_kv_cache *cache, const int32_t *source,
                                      const int32_t *target, int32_t n, void *stream);

/* ---- decode -------------------------------------------------------------------------- */

/* q and out [batch, heads, head_dim] (strides as above), lse [batch, heads]. Query row b is
 * the last token of sequences[b] (NULL = row b of the table) and sees all of its tokens, or
 * with window > 0 the last `window`. The first shared_tokens (a multiple of page_tokens, may
 * be 0) of every sequence in the batch lie in the same pages; they are read once, or by each
 * sequence where that is sooner done. A sequence shorter than that sees what it has, wherever
 * it stands in the batch; a row number outside the table is an empty sequence. max_length
 * bounds every lengths[sequences[b]]; tokens beyond it are not read. (The closer it is, the
 * better the work can be cut; what the page table holds is a bound in any case.) workspace is
 * 16-byte aligned scratch of at least dm_attention_decode_workspace bytes for the same numbers;
 * two calls in flight need two. A page number outside the pool reads as keys and values of zero
 * and sets DM_KV_BAD_TOKEN. */
typedef struct {
  int32_t layer, heads, batch, window;
  int32_t shared_tokens, max_length;
  float scale;
  const void *q;
  void *out;
  float *lse;
  int64_t q_stride[2], out_stride[2];
  const int32_t *sequences;
  void *workspace;
  uint64_t workspace_bytes;
} dm_attention_decode_desc;

DM_API int32_t dm_attention_decode_workspace(const dm_kv_cache *cache, int32_t heads, int32_t batch,
                                             int32_t shared_tokens, int32_t max_length,
                                             uint64_t *bytes);
DM_API int32_t dm_attention_decode(dm_kv_cache *cache, const dm_attention_decode_desc *desc,
                                   void *stream);

#ifdef __cplusplus
}
#endif
#endif
