/*
 * lutmac_kv8.h -- a paged key/value cache held in 8 bits (C ABI): appending
 * rotated keys and values, and attention over it, for sequences of different
 * lengths.
 *
 * The reference keeps one contiguous fp32 cache per model (types.hpp:599-627)
 * and attends it position by position (model.cpp:326-372); this cache takes a
 * quarter of the bytes, so a step that reads long contexts takes a quarter of
 * the time, and its pages are shared by sequences of any lengths.  The decoder
 * (lutmac_decode.h) runs on it when it is created with LMX_KV_INT8.
 *
 * All pointers are DEVICE pointers of the current device, all work is
 * asynchronous on `stream` (NULL = default), nothing is allocated and nothing
 * kept between calls, so calls can be captured into a HIP graph; lengths and
 * page tables are read when the work runs.  Calls that append to a cache and
 * read it must be ordered.
 */
#ifndef LUTMAC_KV8_H
#define LUTMAC_KV8_H

#include <stddef.h>
#include <stdint.h>

#include "lutmac_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define LMX_KV8_PAGE 64   /* tokens of a page */
#define LMX_KV8_BLOCK 16  /* tokens that share a scale (per KV head) */

/* One layer's cache.  value = code * scale of its block, for K and V apart.
 * Token j of a page: key codes k[page][head][j][.], value codes
 * v[page][head][.][j] (transposed, the order the value product reads), scales
 * [page][head][j / 16].  k and v are 16-byte aligned, scales not negative. */
typedef struct {
  int8_t *k;         /* [n_pages][n_kv_heads][64][head_dim] */
  int8_t *v;         /* [n_pages][n_kv_heads][head_dim][64] */
  float *k_scale;    /* [n_pages][n_kv_heads][4] */
  float *v_scale;    /* [n_pages][n_kv_heads][4] */
  size_t n_pages;    /* < 2^31 */
  size_t n_kv_heads; /* 1 .. 512; query heads: 1 .. 64 times as many */
  size_t head_dim;   /* 64 or 128 */
} lmx_kv8_cache;

/* The rows (tokens) of a call and the sequences they belong to: rows
 * offsets[s] .. offsets[s + 1] - 1 are the last of the lengths[s] tokens that
 * sequence s has with them, in order (none: the sequence has no row in this
 * call).  Token j of sequence s lies in page pages[s * max_pages + j / 64].
 * offsets do not decrease; rows below offsets[0] and from offsets[n_seqs] on belong
 * to no sequence and are neither read nor written.  A row whose position is negative (more
 * rows than lengths[s]) or past the table has no place in the cache and sees
 * nothing there; nor has one whose page is outside 0 .. n_pages - 1. */
typedef struct {
  const int32_t *offsets;  /* [n_seqs + 1] */
  const int32_t *lengths;  /* [n_seqs] */
  const int32_t *pages;    /* [n_seqs][max_pages] */
  size_t n_seqs;           /* <= 2^20 */
  size_t max_pages;        /* <= 2^24 */
  size_t n_rows;           /* rows that the row arrays hold, >= offsets[n_seqs]; <= 2^24 */
} lmx_kv8_batch;

/* Rotates and appends: for every row, its keys k and values v (row r at
 * k + r * k_stride, [n_kv_heads][head_dim]) into the cache, the keys rotated to
 * the row's position; its queries q ([n_heads][head_dim]) rotated into q_out
 * (which may be q).  q NULL: keys and values only.  Strides count elements;
 * pointers and strides are multiples of 16 bytes.
 *   rope [rope_positions][head_dim / 2] (cos, sin) pairs turn the pairs (d, d +
 *   head_dim / 2) as the reference's apply_rope does (embedding.cpp:36-75);
 *   NULL: no rotation.  A row at or past rope_positions is left out whole.
 * A block that receives rows gets the scale max(s, amax / 127, 2^-100), s its
 * present scale if it holds earlier tokens of the sequence, amax the largest
 * magnitude of the rows it receives; the codes of its earlier tokens are
 * rounded anew to a scale that has grown.  Scales and codes are those of the
 * rotation and the quotients in 64 bits, rounded once (ties to even), so they
 * do not depend on the order of anything; rotated queries are rounded once
 * from 64 bits (fp32) or from fp32 (16-bit types).  Where a value is not finite the block's
 * scale becomes NaN (as does the attention of every row that sees the block)
 * until the block starts anew.  Blocks are read and written by one workgroup
 * each: the pages that receive rows in one call differ from each other. */
int lmx_kv8_append(const lmx_kv8_cache *cache, const lmx_kv8_batch *batch,
                   int type, const void *k, size_t k_stride, const void *v,
                   size_t v_stride, const void *q, size_t q_stride, void *q_out,
                   size_t q_out_stride, size_t n_heads, const float *rope,
                   size_t rope_positions, void *stream);

/* Bytes of workspace that lmx_kv8_attention needs for a call of these sizes
 * (pointers are not looked at; 0 is possible).  Fewer rows can need more: their
 * pages are split over workgroups. */
int lmx_kv8_attention_workspace(const lmx_kv8_cache *cache,
                                const lmx_kv8_batch *batch, int type,
                                size_t n_heads, size_t *bytes);
/* Attention of the rows' queries (row r at q + r * q_stride, [n_heads]
 * [head_dim], rotated) over their sequences' cached tokens up to their own
 * positions: out = softmax(scale * q . k) v, query head h reading KV head
 * h / (n_heads / n_kv_heads), scale positive.  A row that sees nothing gets zeros.  out
 * (out_stride; elements of `type`) may be q.
 * Products with the codes are exact, sums and softmax statistics fp32.  Before
 * the products queries are rounded to 2^-23 of a power of two above the largest
 * of their head, the weights of the values to 2^-23 of the largest of their page.
 * Large calls of prompts in the 16-bit types hold queries to 2^-39 and weights to
 * 2^-11 of themselves: those where each = ceil(n_rows / n_seqs) * n_heads /
 * n_kv_heads is 96 or more and n_seqs * n_kv_heads * ceil(each / 16) 1024 or more,
 * so that the last bits of a row depend on the call that it is in.  V scales
 * lie between 2^-100 and 2^100; those below 2^-60 of the largest in reach lose
 * bits like the small values of one block do.  A query head with an element
 * that is not finite gives NaN.
 * The work is split by the call's sizes alone, as if its sequences had equal
 * shares of the rows: long prompts and single tokens after long contexts are
 * faster in calls of their own (4096 rows of one sequence and single ones of 63
 * after 8000, 32 + 8 heads of 128, bf16: 722 us together, 164 + 209 apart).
 * workspace: lmx_kv8_attention_workspace bytes, 16-byte aligned, in any state;
 * calls that may overlap in time need workspaces of their own. */
int lmx_kv8_attention(const lmx_kv8_cache *cache, const lmx_kv8_batch *batch,
                      int type, const void *q, size_t q_stride, size_t n_heads,
                      float scale, void *out, size_t out_stride,
                      void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* LUTMAC_KV8_H */
