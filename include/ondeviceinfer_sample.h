/* Choosing tokens from logits with given random numbers.
 *
 * The reference generates greedily only (generation.py:47, :58); this is the
 * call for requests that ask for more, one row of logits each.  Same
 * conventions as ondeviceinfer_wq.h: device pointers, `stream` a hipStream_t
 * (may be NULL), 0 or a WQ_ERR_* code is returned and wq_last_error() holds
 * the message, nothing allocates or synchronizes, and every call may be
 * captured in a HIP graph.
 */
#ifndef ONDEVICEINFER_SAMPLE_H
#define ONDEVICEINFER_SAMPLE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define WQ_LOGITS_F16 0
#define WQ_LOGITS_F32 1

/* Workspace bytes for wq_sample (no initialization needed; calls that may
 * overlap need separate workspaces).  Nearly all of it is a list per row, 8
 * bytes per token of the vocabulary while that comes to at most 64 MiB for all
 * rows, and at least 4096 tokens a row: 64 rows of 151936 take 64 MiB, 65535
 * rows 2 GiB. */
int wq_sample_workspace_size(int64_t rows, int64_t vocab, size_t* bytes);

/* tokens[r] = one token drawn from row r of logits [rows, vocab] (row_stride
 * elements apart) with the uniform number uniform[r] in [0, 1):
 *   order  the tokens by value, the largest first, equal ones by index;
 *   weight w_i = exp((logit_i - largest) / temperature);
 *   top_k  > 0: the first top_k tokens of the order stay;
 *   top_p  < 1: of those, a token stays while the weights before it sum to
 *          less than top_p times the weight of all of those;
 *   min_p  > 0: of those, the ones with w_i >= min_p stay;
 *   the first token of the order always stays.
 * The token is the first of the remaining ones, by index, at which their
 * running weight exceeds uniform[r] times their whole weight.  Weights and
 * sums are 64-bit; those of the tokens within a few octaves of a cut are added
 * as whole numbers of 2^-b of a power of two next to the largest of them, b =
 * 63 - log2(vocab) rounded up and 50 at the most (45 for 151936 tokens).
 * temperature 0 takes the first token of the order.
 * The settings are per-row device arrays; NULL takes the scalar for all rows.
 * A row has no distribution, and its token is -1, when it holds NaN or nothing
 * above -inf, or when its uniform, temperature (negative or not finite), top_p
 * or min_p is no number that has a meaning here (NaN).  Tokens at +inf share
 * the whole weight.  rows <= 65535, vocab <= 2^30. */
int wq_sample(const void* logits, int32_t logits_type, int64_t rows, int64_t vocab, int64_t row_stride,
              const float* uniform, const float* temperature, float temperature_all, const int32_t* top_k,
              int32_t top_k_all, const float* top_p, float top_p_all, const float* min_p, float min_p_all,
              int64_t* tokens, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ONDEVICEINFER_SAMPLE_H */
