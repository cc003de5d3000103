/*
 * hy_rotary.h - C ABI of the B200 (sm_100a) text-decode library: RMS norms of the
 * query and key heads and the position rotation in one pass over their rows, as
 * the decoder does it (rotation, then norm: export/text_decoder_kv.py:66-79) and
 * as the DFlash draft does it (norm, then rotation: export/dflash_export.py). On
 * the way into the paged cache: hy_paged_kv_write_rotated (hy_paged.h).
 *
 * Conventions: those of hy_paged.h (stateless, asynchronous on `stream`, device
 * pointers end in _dev, nothing allocated or kept, calls from several threads may
 * overlap, capturable).
 */
#ifndef HY_ROTARY_H
#define HY_ROTARY_H

#include "hy_decode.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Norms and angles. A head x of a row whose table row has c and s becomes
 *   rotate_first != 0: y = turn(x), y * w / sqrt(mean(y^2) + eps);
 *   rotate_first == 0: turn(x * w / sqrt(mean(x^2) + eps)),
 * turn(x)[d] = x[d] c[d] - x[d + h] s[d], turn(x)[d + h] = x[d + h] c[d + h] + x[d] s[d + h]
 * for d < h = head_dim / 2, in fp32, rounded once. w is q_weight_dev or
 * k_weight_dev. Element d of table row t is at t * table_stride + d of cos_dev and
 * of sin_dev (hy_build_mrope's and hy_rope_value's layout); table rows and weights
 * start on 16 bytes. Row r takes table row positions_dev[r], without positions row
 * r; a row whose table row is not in 0..table_rows - 1 comes out as NaN, and
 * HY_PAGED_BAD_POSITION (hy_paged.h) is set in the status word. */
typedef struct hy_rotation {
    const float* q_weight_dev; /* [head_dim] */
    const float* k_weight_dev; /* [head_dim] */
    const float* cos_dev;      /* (NULL: a table of no rows) */
    const float* sin_dev;
    int table_rows;
    int64_t table_stride;
    const int* positions_dev;  /* [rows], or NULL */
    float eps;                 /* not negative, finite */
    int rotate_first;
} hy_rotation;

/* Row tensors as in hy_paged.h: `rows` rows of q_heads (q) or kv_heads (k) heads of
 * head_dim (64 or 128) elements of `dtype` (HY_DTYPE_F32 or HY_DTYPE_BF16); every
 * (row, head) starts on 16 bytes. The outputs may be the inputs themselves (the
 * same pointer and strides); otherwise they share no memory with the inputs, with
 * each other or with themselves (refused where it shows: rows equally far apart in
 * both, or one row). status_dev (nullable): as in hy_paged_cache.
 * Limits: heads 1024, rows * heads 2^31. */
int hy_norm_rotate(const hy_rotation* rotation, int rows, int q_heads, int kv_heads, int head_dim, int dtype,
                   int device, const void* q_dev, int64_t q_row_stride, int64_t q_head_stride, const void* k_dev,
                   int64_t k_row_stride, int64_t k_head_stride, void* q_out_dev, int64_t q_out_row_stride,
                   int64_t q_out_head_stride, void* k_out_dev, int64_t k_out_row_stride, int64_t k_out_head_stride,
                   int* status_dev, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* HY_ROTARY_H */
