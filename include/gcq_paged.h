/*
 * gcq_paged.h - C ABI of libgcq's paged 4-bit key / value cache: appending rotated keys and values,
 * attention of a ragged batch over the pages, reading rows back. No counterpart in the reference,
 * whose programs keep one contiguous f16 cache per sequence (gcq_set_rows_f16, gcq_flash_attn_ext).
 * Conventions as in gcq.h: 0 / -1 and gcq_last_error(), device pointers, a hipStream_t as void*,
 * arguments checked on the host before anything is launched.
 *
 * A cache is a pool of n_pages pages of page_size tokens, shared by all sequences of one layer. Keys
 * and values are held as Q4_0 blocks of 32 dims: an f16 scale d and 4-bit codes c, value d (c - 8):
 * 1.125 D bytes a token and KV head, where an f16 cache takes 4 D.
 *
 * A batch is n_seq sequences and the new rows (tokens) of each, packed one after the other: sequence
 * s owns rows starts[s] .. starts[s + 1] - 1 (0 <= starts[s] <= starts[s + 1]; no rows is fine). Its
 * row j has position past[s] + j, and position p lives in page pages[s][p / page_size], slot
 * p % page_size. Rows outside every sequence (a batch padded to a fixed size) are left as they are in
 * every output. A page entry outside [0, n_pages), and a position below 0 or past max_pages pages,
 * stands for tokens that are not there: append drops them, attention does not see them, read gives
 * zeros. These arrays live on the device and are read by the kernels: a captured graph follows their
 * contents from replay to replay. Sequences may share pages that a call only reads; two rows of one
 * call that append to the same slot leave some of either's bytes there. A call that takes a launch of 2^32 threads or more (some 2^26 rows) is
 * refused.
 */
#ifndef GCQ_PAGED_H
#define GCQ_PAGED_H

#include "gcq.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    void *  data;        /* gcq_paged_cache_size bytes, 16-byte aligned; any contents to begin with */
    int32_t n_pages;
    int32_t page_size;   /* tokens: 32, 64, 128 or 256 */
    int32_t n_head_kv;
    int32_t head_dim;    /* D: 64, 128 or 256, keys and values alike */
} gcq_paged_cache;

typedef struct {
    const int32_t * pages;  /* [n_seq][max_pages] at row stride ld_pages (elements) */
    int64_t         ld_pages;
    const int32_t * starts; /* [n_seq + 1] */
    const int32_t * past;   /* [n_seq] */
    int32_t         n_seq;
    int32_t         max_pages;
} gcq_paged_batch;

/* Bytes of a cache (0 for a shape that is not supported). */
GCQ_API size_t gcq_paged_cache_size(int n_pages, int page_size, int n_head_kv, int head_dim);

/* Rows of k and v into the cache: k[r][h][d], v[r][h][d] f32 at element strides (k_r, k_h), (v_r, v_h).
 * freqs (n_dims / 2 floats, or NULL: no rotation): the keys' pairs (i, i + n_dims / 2) are turned by
 * position * freqs[i] radians and scaled by attn_factor (ggml_rope_ext's NEOX pairs; freqs[i] =
 * freq_scale base^(-2 i / n_dims) / ff[i]); dims n_dims .. D - 1 pass through. Angle, sine and cosine
 * are taken in 64 bits and a rotated value is rounded once, to 32, whatever the position (gcq_rope_neox
 * keeps ggml's 32-bit angles). Blocks are then encoded as gcq_quantize encodes Q4_0, but for values beyond +-65504
 * (f16's largest), which are taken as that, and NaNs, which are taken as 0: all that the cache holds is finite.
 * q (or NULL) [r][h][d] f32 at (q_r, q_h), n_head heads: rotated alike into q_out [n_rows][n_head][D] f16, what
 * gcq_paged_attn takes. */
GCQ_API int gcq_paged_append(const gcq_paged_cache * cache, const gcq_paged_batch * batch, int64_t n_rows,
                             const float * k, int64_t k_r, int64_t k_h, const float * v, int64_t v_r, int64_t v_h,
                             const float * q, int64_t q_r, int64_t q_h, int n_head, void * q_out, const float * freqs,
                             int n_dims, float attn_factor, void * stream);

/* The values that the cache holds for the batch's rows: k, v [n_rows][n_head_kv][D] f32, 16-byte aligned. past = 0 and all of a
 * sequence's tokens as rows reads the sequence. */
GCQ_API int gcq_paged_read(const gcq_paged_cache * cache, const gcq_paged_batch * batch, int64_t n_rows, float * k,
                           float * v, void * stream);

/* Workspace of gcq_paged_attn for a batch of these sizes (0 for sizes it rejects). */
GCQ_API size_t gcq_paged_attn_workspace(const gcq_paged_cache * cache, const gcq_paged_batch * batch, int64_t n_rows,
                                        int n_head, int64_t max_rows);
/* out[r][h] = sum over the keys j that row r sees of softmax_j(scale q[r][h] . K[j]) V[j], its rows appended before:
 * a row at position p sees the keys 0 .. p of its sequence, with window > 0 the last `window` of them; no key: zeros.
 * q f16 [r][h][D] at element strides (q_r, q_h), multiples of 8; out f32 [n_rows][n_head][D]; n_head a multiple of
 * n_head_kv, KV head h * n_head_kv / n_head. Scores, sums and outputs are f32's; a weight is held to 2^-23 of itself,
 * but no finer than 2^-35 of the row's largest (smaller ones come to 0). A query with a NaN or an infinity gives NaNs
 * where it sees a key. max_rows: no sequence has more rows than this (rows past it are left as they are); n_rows where
 * nothing is known. ws: gcq_paged_attn_workspace bytes, 256-byte aligned, any contents; calls
 * that can overlap need one each. */
GCQ_API int gcq_paged_attn(const gcq_paged_cache * cache, const gcq_paged_batch * batch, int64_t n_rows, const void * q,
                           int64_t q_r, int64_t q_h, int n_head, int64_t max_rows, int window, float scale, float * out,
                           void * ws, size_t ws_size, void * stream);

#ifdef __cplusplus
}
#endif

#endif /* GCQ_PAGED_H */
