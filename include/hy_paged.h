/*
 * hy_paged.h - C ABI of the paged KV cache of the B200 (sm_100a) text-decode
 * library: K / V rows written into pages (quantised as they are written),
 * read back, and attended to by new rows (one token, a verify block, a chunk
 * of a prompt) of several sequences at once, optionally through a sliding
 * window with sinks. No reference counterpart for the pages; the attention is
 * PreciseSDPA's (src/precise_sdpa.cpp:281-329) and the append
 * append_or_grow_kv_cache's (src/kv_cache_capacity.cpp:232-280), over pages.
 *
 * Conventions: those of hy_decode.h (int status, hy_last_error()), except
 *   - these calls need no hy_ctx. They run asynchronously on `stream`
 *     (a cudaStream_t of the cache's device; NULL: the default stream) and can
 *     be captured into a graph; the calling thread's current device is left as
 *     it was;
 *   - they allocate nothing and keep nothing between calls: all memory is the
 *     caller's, names ending in _dev are device pointers. Calls from several
 *     threads may overlap; calls that run at the same time need a workspace
 *     each and must not write the same cache rows, rows or status;
 *   - lengths, row ranges and page numbers are read on the device, so a
 *     captured call follows what those arrays hold when it is replayed.
 */
#ifndef HY_PAGED_H
#define HY_PAGED_H

#include "hy_decode.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Cache types beside HY_DTYPE_F32 and HY_DTYPE_BF16, with one fp32 scale per
 * row and head: a value is code * scale (a caller's own scales may have
 * either sign). */
enum hy_paged_dtype { HY_DTYPE_E4M3 = 2, HY_DTYPE_INT8 = 3 };

/* Bits that the kernels set in *status_dev (never cleared by the library) when
 * the arrays on the device do not hold; the offending part is skipped. */
enum hy_paged_status {
    HY_PAGED_BAD_PAGE = 1,   /* page number outside the cache: its rows are not written, stay as they were
                                in what is read back, and are not seen by attention */
    HY_PAGED_BAD_LENGTH = 2, /* kv_len negative or beyond table_width * page_size: the sequence is left out */
    HY_PAGED_BAD_ROWS = 4,   /* q_start not ascending or outside the rows: the sequence is left out */
    HY_PAGED_TIMEOUT = 8     /* a bounded wait inside a kernel gave up */
};

/* Element d of (page, head, row) is at page * page_stride + head * head_stride
 * + row * row_stride + d of k_dev and of v_dev, its scale (8-bit types) at
 * page * scale_page_stride + head * scale_head_stride + row * scale_row_stride.
 * Strides are in elements, not negative; k_dev, v_dev and every row start on
 * 16 bytes. E4M3 codes are finite (hy_paged_kv_write writes no others). */
typedef struct hy_paged_cache {
    int dtype;        /* HY_DTYPE_F32, _BF16, _E4M3 or _INT8 */
    int num_pages;
    int num_kv_heads;
    int page_size;    /* rows of a page, any number from 1 */
    int head_dim;     /* 64 or 128 */
    int device;
    void* k_dev;
    void* v_dev;
    int64_t page_stride, head_stride, row_stride;
    float* k_scale_dev; /* NULL for F32 and BF16 */
    float* v_scale_dev;
    int64_t scale_page_stride, scale_head_stride, scale_row_stride;
    int* status_dev;    /* nullable; hy_paged_status bits */
} hy_paged_cache;

/* The batch's sequences. Sequence s has the rows [q_start[s], q_start[s + 1])
 * of the row tensors and kv_len[s] positions in the cache, of which its n rows
 * are the last: its row i stands at position kv_len[s] - n + i (rows before
 * position 0, where kv_len[s] < n, are padding: not written, not read, and
 * attending to nothing). Position p lives in row p % page_size of page
 * block_table[s * table_stride + p / page_size]. Rows outside every sequence's
 * range are left as they were. Sequences may share pages that are only read;
 * a row of a page written twice in one call keeps neither value for certain. */
typedef struct hy_paged_batch {
    int num_seqs;
    int max_rows;              /* about the most rows of a sequence: attention is laid out for
                                  it, all sequences alike (another number costs time, not
                                  correctness; tokens beside long chunks are faster in a
                                  call of their own) */
    int table_width;
    int64_t table_stride;
    const int* q_start_dev;    /* [num_seqs + 1] */
    const int* kv_len_dev;     /* [num_seqs] */
    const int* block_table_dev;
} hy_paged_batch;

/* Row tensors: `rows` rows of num_kv_heads (k, v) or q_heads (q, out) heads of
 * head_dim elements of `dtype` (HY_DTYPE_F32 or HY_DTYPE_BF16), element d of
 * (row, head) at row * row_stride + head * head_stride + d; every (row, head)
 * starts on 16 bytes, and those that a call writes share no memory. */

/* Writes k and v of every row at its position. F32 and BF16 caches: rounded to
 * nearest. 8-bit caches: scale = max(max|x| / M, 2^-126) in fp32 with M = 448
 * (E4M3) or 127 (INT8), code = x / scale rounded to the nearest code, ties to
 * even (the quotient is exact). A (row, head) that holds an infinity or a NaN
 * gets the scale NaN and codes 0: it reads as NaN. */
int hy_paged_kv_write(const hy_paged_cache* cache, const hy_paged_batch* batch, int rows, int dtype,
                      const void* k_dev, int64_t k_row_stride, int64_t k_head_stride, const void* v_dev,
                      int64_t v_row_stride, int64_t v_head_stride, void* stream);
/* Reads the same positions back: row i of sequence s gets position
 * kv_len[s] - n + i (n = kv_len[s] reads whole sequences). code * scale in
 * fp32, then rounded to `dtype`. */
int hy_paged_kv_read(const hy_paged_cache* cache, const hy_paged_batch* batch, int rows, int dtype, void* k_dev,
                     int64_t k_row_stride, int64_t k_head_stride, void* v_dev, int64_t v_row_stride,
                     int64_t v_head_stride, void* stream);

/* Attention of the batch's rows over the cache, which holds the rows' own keys
 * and values already: out = softmax(scale * q k^T) v over the visible
 * positions. Query head h reads KV head h / (q_heads / num_kv_heads). A row at
 * position p sees position j when
 *   causal != 0: j <= p, and with window > 0 also p - j < window or j < sinks;
 *   causal == 0: every j < kv_len (window must be 0).
 * A row that sees nothing gives zeros. Positions that a row does not see do
 * not reach its output, whatever they hold (infinities and NaN included).
 * scale must be positive, and scale * log2(e) finite. q and out have the same
 * dtype and must not overlap. Products and sums are in fp32 (BF16 rows: as the
 * tensor cores add, which cut sums instead of rounding them).
 * F32 rows: products are exact to 2^-21. Over 8-bit caches q and the weights
 * (probabilities times v's scale) are off by 2^-22 of themselves, or by 2^-39 of
 * a row's largest where that is more.
 * BF16 rows: probabilities are rounded to bf16 before they multiply v; over
 * 8-bit caches they are multiplied by v's scale and rounded to f16, off by 2^-11
 * of themselves, or by 2^-39 of the row's largest such product (2^-27 where
 * max_rows times q_heads / num_kv_heads is above 32) where that is more.
 * Over 8-bit caches scales of v beyond 2^100 overflow and those below 2^-100
 * lose bits. An infinity that a row does see may give NaN.
 * Limits: q_heads and num_kv_heads 1024, num_seqs 65535, rows * q_heads 2^31,
 * table_width * page_size 2^30; writes and reads take row and head strides
 * (the cache's head strides too) below 2^31. */
int hy_paged_attention(const hy_paged_cache* cache, const hy_paged_batch* batch, int rows, int q_heads, int dtype,
                       const void* q_dev, int64_t q_row_stride, int64_t q_head_stride, void* out_dev,
                       int64_t out_row_stride, int64_t out_head_stride, float scale, int causal, int window,
                       int sinks, void* workspace_dev, size_t workspace_bytes, void* stream);
/* Bytes of workspace_dev (16-byte aligned, any contents) that the call needs.
 * They do not depend on the sequences' lengths. */
int hy_paged_attention_workspace(const hy_paged_cache* cache, const hy_paged_batch* batch, int rows, int q_heads,
                                 int dtype, size_t* bytes);

#ifdef __cplusplus
}
#endif

#endif /* HY_PAGED_H */
