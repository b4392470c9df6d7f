/*
 * lutmac_verify.h -- verification of drafted tokens (C ABI): which of the tokens
 * that a cheaper model proposed a program keeps, and the token that follows them, so
 * that what comes out is distributed as if every token had been sampled from the
 * target model whose logits are given (what a cache makes of tokens that were
 * dropped again: lmx_kv8_trim).
 *
 * The reference samples one token at a time from its logits (Model::sample,
 * src/model.cpp:455-490); this is the same choice for several positions of many
 * sequences at once, with the random numbers given.
 *
 * All pointers are DEVICE pointers of the current device, all work is asynchronous
 * on `stream` (NULL = default), nothing is allocated and nothing kept between
 * calls, so calls can be captured into a HIP graph.
 */
#ifndef LUTMAC_VERIFY_H
#define LUTMAC_VERIFY_H

#include <stddef.h>
#include <stdint.h>

#include "lutmac_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Rows offsets[s] .. offsets[s + 1] - 1 of a call are sequence s's: row by row the
 * target's logits, drafts[r] the token drafted at row r (the last row of a sequence has none: its entry
 * is not looked at), so a sequence with n drafted tokens has n + 1 rows.
 * Offsets do not decrease; rows of no sequence reach nothing and their tokens stay. */
typedef struct {
  const int32_t *offsets;   /* [n_seqs + 1] */
  const int32_t *drafts;    /* [n_rows] */
  const float *uniforms;    /* [n_rows][2], each 0 <= u < 1 */
  const float *temperature; /* [n_seqs], or NULL: 1 */
  size_t n_seqs;            /* <= 2^20 */
  size_t n_rows;            /* rows that the row arrays hold, >= offsets[n_seqs]; <= 2^20 */
  size_t vocab;             /* 1 .. 2^24 */
} lmx_drafts;

/* Bytes of workspace that lmx_verify_drafts needs for a call of these sizes
 * (pointers are not looked at). */
int lmx_verify_drafts_workspace(const lmx_drafts *d, int type, size_t *bytes);
/* With p = softmax(logits[r] / temperature) and q = probs[r], the draft's
 * probabilities (probs NULL: q is 1 for the drafted token, 0 else), the drafted
 * token t of row r is accepted if u0 q[t] < p[t] for (u0, u1) = uniforms[r].  The
 * first row where it is not ends its sequence with a token sampled from max(0, p - q)
 * (from p, if that is 0 everywhere); if all are, the last row does, from p.  The token sampled is the first
 * whose weights with those of the tokens before it exceed u1 times the sum of all.
 *   accepted [n_seqs]: drafted tokens kept; tokens [n_rows]: row by row the
 *   accepted tokens, then the sampled one, then -1.  (No rows: 0 and nothing.)
 * A drafted token outside 0 .. vocab - 1 is not accepted, but it is no mark of
 * "nothing drafted": the token is sampled from max(0, p - q) of the row's probs all
 * the same (probs NULL: from p).  A sequence with fewer drafts has fewer rows.
 * A temperature of 0 (or below, or NaN) is the limit: p is 1 for the first of the
 * largest logits.  Logits of -inf have p = 0; a row whose logits are all -inf,
 * or with a NaN or +inf, accepts nothing and gives the token -1.  Everything is summed
 * and compared in 64 bits from the given numbers, each e^x to 2^-44 of itself, so
 * that tokens are those of exact arithmetic, and do not depend on how sums are ordered, but where a
 * number is within some 2^-40 of a border.
 * logits: elements of `type`, row r at logits + r * stride (elements; at least
 * vocab), aligned to an element; probs fp32, row r at probs + r * probs_stride.
 * accepted and tokens overlap no input.
 * workspace: lmx_verify_drafts_workspace bytes, 16-byte aligned, in any state;
 * calls that may overlap in time need workspaces of their own. */
int lmx_verify_drafts(const lmx_drafts *d, int type, const void *logits, size_t stride,
                      const float *probs, size_t probs_stride, int32_t *accepted,
                      int32_t *tokens, void *workspace, size_t workspace_bytes,
                      void *stream);

#ifdef __cplusplus
}
#endif
#endif /* LUTMAC_VERIFY_H */
