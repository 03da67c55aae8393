/*
 * gcq_draft.h - C ABI of libgcq's steps with drafted tokens over the paged cache (gcq_paged.h): a tree of guesses for each
 * sequence is appended, attended and verified in one pass of the model, then its accepted rows are moved together. No
 * counterpart in the reference, which decodes a token at a time. Conventions as in gcq_paged.h; batches as there.
 *
 * A sequence's new rows are a tree: row 0 is its last accepted token, whose keys and values are not in the cache yet, every
 * other row a guess at what follows an earlier one. parents [n_rows]: the number, within the sequence, of the row that a row
 * follows; anything but an earlier row's number (-1) is taken as none: the row follows the cached tokens. Row j lies in the
 * cache at slot past + j, as in any batch. Its depth is 0 without a parent and one more than its parent's with one, its
 * position past + depth, and it sees the slots below past, its ancestors and itself. A chain (parents j - 1) is an ordinary
 * batch. At most 1024 rows a sequence.
 *
 * A step: gcq_draft_tree, then for each layer gcq_paged_append_at and gcq_paged_attn_tree, then gcq_draft_verify on the last
 * layer's logits, and gcq_paged_move for all layers; past grows by count[s], the last of tokens[s] is the next step's row 0.
 */
#ifndef GCQ_DRAFT_H
#define GCQ_DRAFT_H

#include "gcq_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

#define GCQ_DRAFT_MAX_ROWS 1024

/* Positions and masks of a batch's trees, once for a step: positions[r] = past + depth; mask [n_rows][ld_mask], bit i % 32 of
 * word i / 32: the row sees row i of its sequence. window > 0: only rows that are less than `window` positions back. max_rows:
 * no sequence has more rows than this (rows past it, and rows of no sequence, are left as they are); 32 ld_mask >= max_rows or
 * n_rows, ld_mask <= 32. Of the batch, starts and past are read. */
GCQ_API int gcq_draft_tree(const gcq_paged_batch * batch, int64_t n_rows, const int32_t * parents, int64_t max_rows,
                           int window, int32_t * positions, uint32_t * mask, int64_t ld_mask, void * stream);

/* gcq_paged_append with positions [n_rows] that are not the rows' slots: row j of a sequence still goes to slot past + j, and is
 * turned by positions[r] * freqs[i]. Of trees, of rows behind a prompt of which a part was left out, .. */
GCQ_API int gcq_paged_append_at(const gcq_paged_cache * cache, const gcq_paged_batch * batch, int64_t n_rows,
                                const int32_t * positions, const float * k, int64_t k_r, int64_t k_h, const float * v,
                                int64_t v_r, int64_t v_h, const float * q, int64_t q_r, int64_t q_h, int n_head, void * q_out,
                                const float * freqs, int n_dims, float attn_factor, void * stream);

/* gcq_paged_attn of rows that see the slots below past and, of the sequence's new rows, those of their mask (any mask of rows
 * that were appended before, a tree's or not; bits past the sequence's rows count as 0). window > 0: of the slots below past,
 * those above positions[r] - window (positions below past count as past; not read without a window); the mask's own window is
 * gcq_draft_tree's. A row that sees nothing gives zeros; what no row sees may hold anything. mask [n_rows][ld_mask],
 * ld_mask <= 32; max_rows <= 1024 unless n_rows is less. Workspace: gcq_paged_attn_workspace. */
GCQ_API int gcq_paged_attn_tree(const gcq_paged_cache * cache, const gcq_paged_batch * batch, int64_t n_rows,
                                const int32_t * positions, const uint32_t * mask, int64_t ld_mask, const void * q, int64_t q_r,
                                int64_t q_h, int n_head, int64_t max_rows, int window, float scale, float * out, void * ws,
                                size_t ws_size, void * stream);

/* Workspace of gcq_draft_verify (0 for sizes it rejects). */
GCQ_API size_t gcq_draft_verify_workspace(int n_seq, int64_t n_rows, int64_t n_vocab, int64_t max_rows);
/* Which drafts stand, and the token after them, so that all tokens are distributed as if drawn from the target one by one.
 * Row r of a tree has token tokens[r], the target's logits (row r of logits, stride ld) for what follows it, and coins[r], a
 * uniform random number of [0, 1). p = softmax(logits / temperature[s]) (temperature NULL: 1).
 *   With draft_logits: a row's children were drawn, independently of each other, from q = softmax(draft_logits / temperature),
 *   row r's for what follows r (not read where a row has no children). From the root on, a row's children are looked at in
 *   order: child i stands if coin_i < r(t_i) / q(t_i), r = p at first; if it falls r becomes max(r - q, 0), normalised.
 *   draft_logits NULL: children are guesses that were not drawn: child i stands if coin_i < r(t_i); if it falls r loses t_i and is
 *   normalised.
 * The first child that stands is the next row; where none does, the next token is drawn from r with row 0's coin: the lowest token
 * whose cumulative sum is above coin times the sum. Temperature 0 (or less, or a NaN): a child stands if it is the
 * target's largest logit (the lowest of equals), which is the next token where none does. All in 64 bits from the f32
 * logits on, the exponentials to 2^-43 of themselves. A logit that is a NaN counts as -inf (never drawn), +inf as the largest float; where a row's logits are all
 * -inf nothing follows: the token is -1. A draft outside [0, n_vocab) falls, with draft_logits as a draw from q does that fell; it
 * was none, and what follows it is not distributed as the target: rows that fill a tree up to a fixed size have no parent
 * (-1) instead, and are not looked at, whatever else they hold. (Where rounding leaves r nothing, it is p.)
 * Results, ints, for sequence s: count[s], the rows that stand, the root among them (0: no rows); rows [n_seq][max_path] their
 * numbers within the sequence, -1 from count on; tokens_out [n_seq][max_path] the token that follows each: the next row's, for
 * the last one the drawn one. A path ends after max_path rows. Rows past max_rows of a sequence are not looked at. ws:
 * gcq_draft_verify_workspace bytes, 256-byte aligned, any contents; calls that can overlap need one each. */
GCQ_API int gcq_draft_verify(const int32_t * starts, int n_seq, int64_t n_rows, const int32_t * parents,
                             const int32_t * tokens, const float * logits, int64_t ld, const float * draft_logits,
                             int64_t draft_ld, int64_t n_vocab, const float * temperature, const float * coins,
                             int64_t max_rows, int max_path, int32_t * count, int32_t * rows, int32_t * tokens_out, void * ws,
                             size_t ws_size, void * stream);

/* In each of n_caches caches of one shape, slot past[s] + i takes what slot past[s] + rows[s][i] holds, for i < count[s] and
 * i < max_keep; rows [n_seq][ld_rows]. All sources as they were before the call. An entry below its own number i, and one
 * whose slots are not there, moves nothing (a path's rows are all at or above their numbers). Of the batch, pages and past are
 * read. caches: an array of pointers, on the host, to caches that share no memory. */
GCQ_API int gcq_paged_move(const gcq_paged_cache * const * caches, int n_caches, const gcq_paged_batch * batch,
                           const int32_t * count, const int32_t * rows, int64_t ld_rows, int max_keep, void * stream);

#ifdef __cplusplus
}
#endif

#endif /* GCQ_DRAFT_H */
