/* Operators over a paged key/value cache: many sequences at once.
 *
 * The reference's cache holds one contiguous [batch, kv_heads, max_seq, 128]
 * tensor per layer and one length for the whole batch (cache.py:22-92); here
 * the keys and values of any number of sequences of different lengths lie in
 * pages of one pool per layer, and a sequence is a row of page numbers.
 *
 *   key/value_pages [num_pages, kv_heads, page_size, 128] fp16, the last three
 *                   dimensions contiguous, page p at p * *_page_stride
 *                   elements; page_size % 16 == 0
 *   page_table      [sequences, table_width] int32 (rows contiguous): position
 *                   i of sequence b is row i % page_size of page
 *                   page_table[b, i / page_size]
 *   query_starts    [sequences + 1] int32, non-decreasing: the call's tokens
 *                   query_starts[b] .. query_starts[b + 1] - 1 are the newest
 *                   ones of sequence b (possibly none)
 *   seq_lens        [sequences] int32: the positions of sequence b, its new
 *                   tokens included
 *
 * All three are read on the device, so a captured graph follows them.  Tokens
 * behind query_starts[sequences] (padding) and tokens of a sequence whose
 * starts are not 0 <= start <= end <= tokens are left as they were; table
 * entries behind a sequence's length are never read.  Same conventions
 * otherwise as ondeviceinfer_wq.h: device pointers, fp16 as uint16_t, `stream`
 * a hipStream_t (may be NULL), 0 or a WQ_ERR_* code is returned and
 * wq_last_error() holds the message, nothing allocates or synchronizes, and
 * every call may be captured in a HIP graph.
 */
#ifndef ONDEVICEINFER_PAGED_H
#define ONDEVICEINFER_PAGED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Per-head q/k RMSNorm and the position rotation of the new tokens, k and v
 * into their pages.
 *   qkv          [tokens, q_heads*128 | kv_heads*128 | kv_heads*128]
 *   q/k_norm     per-head RMSNorm weights [128] (NULL: no norm)
 *   cos/sin      rotation tables [table_positions, 128] fp16
 *   positions    [tokens] int32 row of the tables for each token (drafted
 *                tokens of a tree), NULL: the token's index in its sequence
 *   q_out        [tokens, q_heads, 128] the normalized, rotated queries; must
 *                not overlap qkv
 * y = u * cos + rotate_half(u) * sin with u = x * rsqrt(mean(x^2) + eps) * w,
 * in fp32 and rounded to fp16 once.  A token whose index has no page (a
 * negative index, one past the table's width, a page number outside the pool)
 * or whose position is outside the tables gets NaN in q_out and writes
 * nothing to the pages.  Of two tokens that name the same page row either's
 * elements are left there, eight at a time.
 * Replaces, for a batch: q/k rms_norm + apply_rotary_pos_emb + cache.update
 * (quantized_model.py:177-195, layers.py:64-80, cache.py:60-80). */
int wq_paged_append(const uint16_t* qkv, int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                    const uint16_t* q_norm_weight, const uint16_t* k_norm_weight, float eps,
                    const uint16_t* cos_table, const uint16_t* sin_table, int64_t table_positions,
                    const int32_t* positions, const int32_t* page_table, int64_t table_width,
                    const int32_t* query_starts, const int32_t* seq_lens, int64_t sequences, uint16_t* key_pages,
                    int64_t key_page_stride, uint16_t* value_pages, int64_t value_page_stride, int64_t num_pages,
                    int64_t page_size, uint16_t* q_out, void* stream);

/* Workspace bytes for wq_paged_attention (0: none).  It holds the partial
 * results of sequences split over workgroups between the attention launch and
 * its merge; it needs no initialization, and calls that may overlap need
 * separate workspaces. */
int wq_paged_attention_workspace_size(int64_t tokens, int64_t sequences, int64_t q_heads, int64_t kv_heads,
                                      int64_t head_dim, int64_t table_width, int64_t page_size, size_t* bytes);

/* Grouped-query attention of the new tokens over their sequences' pages
 * (which hold the new tokens' keys and values already).
 *   q, out       [tokens, q_heads, 128] fp16, token-major; out may be q itself
 *                and must not overlap it otherwise
 *   tree_mask    NULL: token i of a sequence attends its positions up to its
 *                own.  Otherwise [tokens] int64: the new tokens are drafted
 *                ones that form a tree, every one attends all positions
 *                before them and, of the sequence's new tokens, those whose
 *                bit is set in its mask (bit j: the j-th, its own bit
 *                included); at most 64 new tokens per sequence.
 * out = softmax(scale * q . k) . v in fp32, the probabilities rounded to fp16
 * for the product with v and their sum: by 2^-11 of each, or by 2^-36 of the
 * largest of its chunk of keys where that is more.  What a token does not attend has no influence on
 * it, infinite or NaN as it may be; one that attends an infinite or NaN value
 * is no number there, and may be NaN in its other elements too.  A token that
 * attends nothing gets zeros, one that
 * attends a position without a page (past the table's width, a page number
 * outside the pool) NaN, and so do all tokens of a sequence with more than 64
 * drafted ones.  scale must be positive and finite, q_heads / kv_heads <= 16.
 * Replaces, for a batch: F.scaled_dot_product_attention over the cached keys
 * (attention.py:35-85, quantized_model.py:186-199). */
int wq_paged_attention(const uint16_t* q, int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                       const uint16_t* key_pages, int64_t key_page_stride, const uint16_t* value_pages,
                       int64_t value_page_stride, int64_t num_pages, int64_t page_size, const int32_t* page_table,
                       int64_t table_width, const int32_t* query_starts, const int32_t* seq_lens, int64_t sequences,
                       const int64_t* tree_mask, float scale, uint16_t* out, void* workspace, size_t workspace_bytes,
                       void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ONDEVICEINFER_PAGED_H */
