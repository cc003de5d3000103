/*
 * hy_logprobs.h - C ABI of the B200 (sm_100a) text-decode library: log
 * probabilities of given tokens, the entropy and the most likely alternatives of
 * rows of logits. Beside the LM head's selection (hy_lm_head_select, hy_decode.h),
 * which gives the argmax alone; hy_lm_head_logprobs runs it behind a context's LM
 * head. No reference counterpart.
 *
 * Conventions: those of hy_paged.h (stateless, asynchronous on `stream`, device
 * pointers end in _dev, nothing allocated or kept, calls from several threads may
 * overlap, capturable).
 */
#ifndef HY_LOGPROBS_H
#define HY_LOGPROBS_H

#include "hy_decode.h"

#ifdef __cplusplus
extern "C" {
#endif

#define HY_LOGPROBS_MAX_TOP 64

/* Logits x [rows x vocab] of `dtype` (HY_DTYPE_F32 or HY_DTYPE_BF16), element v of
 * row r at r * row_stride + v (any alignment of a row). With lse = log sum exp(x):
 *   logprobs_dev [rows x tokens_per_row] = x[token] - lse for the row's tokens
 *     (NaN for a token outside 0 .. vocab - 1);
 *   entropy_dev [rows] (nullable) = lse - sum of p x, p = exp(x - lse);
 *   top_ids_dev, top_logprobs_dev [rows x top] = the `top` largest logits' tokens,
 *     largest first, of equal ones the lower token first, and their x - lse; where
 *     fewer are above -infinity, -1 and -infinity follow.
 * Logits of -infinity (masked tokens) have probability 0. A row that holds a NaN or
 * +infinity, or nothing above -infinity, gives NaN throughout and tokens of -1. All
 * in fp32; what is left beside a probability near 1 keeps its relative precision.
 * 0 <= top <= HY_LOGPROBS_MAX_TOP, top <= vocab, vocab <= 2^20, tokens_per_row <=
 * 2^30, rows * max(tokens_per_row, top, 8) < 2^31 (a row has up to 8 blocks). */
int hy_token_logprobs(const void* logits_dev, int rows, int vocab, int64_t row_stride, int dtype, int device,
                      const int* tokens_dev, int tokens_per_row, int top, float* logprobs_dev, float* entropy_dev,
                      int* top_ids_dev, float* top_logprobs_dev, void* stream);

/* The same behind a context's LM head: logits of `rows` (1..16) final-normed hidden
 * rows [rows x 1024] (run_lm_head, src/text_runtime.cpp:430-439, no repetition
 * penalty), host buffers. tokens [rows] (nullable with logprobs), entropy,
 * top_ids / top_logprobs [rows x top] nullable (top 0). */
int hy_lm_head_logprobs(hy_ctx* ctx, const float* hidden, int rows, const int* tokens, int top, float* logprobs,
                        float* entropy, int* top_ids, float* top_logprobs);

#ifdef __cplusplus
}
#endif

#endif /* HY_LOGPROBS_H */
