// Host side of the stateless calls: errors, checks of arguments, the device of a
// call, the device's view of a cache and a batch. Every check needs no device.
#pragma once

#include <cuda_runtime.h>

#include <climits>
#include <cstdio>
#include <string>

#include "hy_paged.cuh"
#include "hy_paged.h"

namespace hy_internal {
void set_last_error(const std::string& msg);
}  // namespace hy_internal

namespace hy {

inline int fail(int code, const char* msg) noexcept
{
    try
    {
        hy_internal::set_last_error(msg);
    }
    catch (...)   // no memory for the message: the status still tells
    {
    }
    return code;
}

inline int cuda_fail(const char* what, cudaError_t e) noexcept
{
    char msg[256];
    snprintf(msg, sizeof msg, "%s: %s", what, cudaGetErrorString(e));
    return fail(e == cudaErrorMemoryAllocation ? HY_ERR_OUT_OF_MEMORY : HY_ERR_CUDA, msg);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// log2 of n where it is one, else -1.
inline int power_of_two(int n)
{
    if (n & (n - 1)) return -1;
    int s = 0;
    while ((1 << s) < n) ++s;
    return s;
}

// A stride of a dimension with one entry is never taken.
inline bool off16(long long stride, int elem, int entries) { return entries > 1 && stride * elem % 16 != 0; }

inline int elem_size(int dtype) { return dtype == HY_DTYPE_F32 ? 4 : dtype == HY_DTYPE_BF16 ? 2 : 1; }

inline int check_cache(const hy_paged_cache* c)
{
    if (!c) return fail(HY_ERR_INVALID_ARGUMENT, "cache is null");
    if (c->dtype < HY_DTYPE_F32 || c->dtype > HY_DTYPE_INT8)
        return fail(HY_ERR_INVALID_ARGUMENT, "cache dtype must be F32, BF16, E4M3 or INT8");
    if (c->head_dim != 64 && c->head_dim != 128)
        return fail(HY_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
    if (c->num_pages < 1 || c->page_size < 1 || c->num_kv_heads < 1)
        return fail(HY_ERR_INVALID_ARGUMENT, "num_pages, page_size and num_kv_heads must be positive");
    if (c->num_kv_heads > 1024) return fail(HY_ERR_UNSUPPORTED, "num_kv_heads must be at most 1024");
    if (!c->k_dev || !c->v_dev) return fail(HY_ERR_INVALID_ARGUMENT, "cache memory is null");
    const int e = elem_size(c->dtype);
    if (!aligned16(c->k_dev) || !aligned16(c->v_dev) || off16(c->page_stride, e, c->num_pages) ||
        off16(c->head_stride, e, c->num_kv_heads) || off16(c->row_stride, e, c->page_size))
        return fail(HY_ERR_INVALID_ARGUMENT, "cache rows must start on 16 bytes");
    if (c->page_stride < 0 || c->head_stride < 0 || c->row_stride < 0 || c->scale_page_stride < 0 ||
        c->scale_head_stride < 0 || c->scale_row_stride < 0)
        return fail(HY_ERR_INVALID_ARGUMENT, "cache strides must not be negative");
    const bool codes = e == 1;
    if (codes && (!c->k_scale_dev || !c->v_scale_dev))
        return fail(HY_ERR_INVALID_ARGUMENT, "an 8-bit cache needs k and v scales");
    if (!codes && (c->k_scale_dev || c->v_scale_dev))
        return fail(HY_ERR_INVALID_ARGUMENT, "scales belong to 8-bit caches only");
    if (c->device < 0) return fail(HY_ERR_INVALID_ARGUMENT, "device must not be negative");
    return HY_OK;
}

inline int check_batch(const hy_paged_batch* b, const hy_paged_cache* c)
{
    if (!b) return fail(HY_ERR_INVALID_ARGUMENT, "batch is null");
    if (b->num_seqs < 0 || b->num_seqs > 65535) return fail(HY_ERR_INVALID_ARGUMENT, "num_seqs must be in 0..65535");
    if (b->max_rows < 0) return fail(HY_ERR_INVALID_ARGUMENT, "max_rows must not be negative");
    if (b->num_seqs == 0) return HY_OK;
    if (b->table_width < 0 || b->table_stride < 0)
        return fail(HY_ERR_INVALID_ARGUMENT, "table_width and table_stride must not be negative");
    if (static_cast<long long>(b->table_width) * c->page_size > INT_MAX / 2)
        return fail(HY_ERR_CAPACITY, "table_width * page_size must be below 2^30");
    if (!b->q_start_dev || !b->kv_len_dev || (b->table_width > 0 && !b->block_table_dev))
        return fail(HY_ERR_INVALID_ARGUMENT, "batch arrays are null");
    return HY_OK;
}

inline int check_rows(const char* name, const void* p, int rows, int heads, long long row_stride, long long head_stride, int dtype)
{
    char msg[96];
    const int e = elem_size(dtype);
    const char* what = !p                                                                      ? "%s is null"
                       : row_stride < 0 || head_stride < 0                                     ? "%s strides must not be negative"
                       : !aligned16(p) || off16(row_stride, e, rows) || off16(head_stride, e, heads) ? "%s rows must start on 16 bytes"
                                                                                               : nullptr;
    if (!what) return HY_OK;
    snprintf(msg, sizeof msg, what, name);
    return fail(HY_ERR_INVALID_ARGUMENT, msg);
}

// Rows that a call writes: entries of a dimension whose stride is below head_dim share elements for certain.
inline int check_apart(const char* name, int rows, int heads, int head_dim, long long row_stride, long long head_stride)
{
    if ((rows < 2 || row_stride >= head_dim) && (heads < 2 || head_stride >= head_dim)) return HY_OK;
    char msg[96];
    snprintf(msg, sizeof msg, "%s rows must not overlap", name);
    return fail(HY_ERR_INVALID_ARGUMENT, msg);
}

inline int check_dtype(int rows, int dtype)
{
    if (rows < 0) return fail(HY_ERR_INVALID_ARGUMENT, "rows must not be negative");
    if (dtype != HY_DTYPE_F32 && dtype != HY_DTYPE_BF16)
        return fail(HY_ERR_INVALID_ARGUMENT, "row dtype must be F32 or BF16");
    return HY_OK;
}

// The cache's device for the length of a call.
class DeviceGuard {
public:
    explicit DeviceGuard(int device)
    {
        error_ = cudaGetDevice(&before_);
        if (error_ == cudaSuccess && before_ != device)
        {
            error_ = cudaSetDevice(device);
            restore_ = error_ == cudaSuccess;
        }
    }
    ~DeviceGuard()
    {
        if (restore_) cudaSetDevice(before_);
    }
    cudaError_t error() const { return error_; }

private:
    int before_ = 0;
    bool restore_ = false;
    cudaError_t error_;
};

inline PagedCache device_cache(const hy_paged_cache* c)
{
    return {c->k_dev, c->v_dev, c->k_scale_dev, c->v_scale_dev, c->page_stride, c->head_stride, c->row_stride,
            c->scale_page_stride, c->scale_head_stride, c->scale_row_stride, c->num_pages, c->page_size,
            c->num_kv_heads, c->status_dev};
}

inline PagedBatch device_batch(const hy_paged_batch* b, int rows)
{
    return {b->q_start_dev, b->kv_len_dev, b->block_table_dev, b->table_stride, b->table_width, b->num_seqs, rows};
}

inline int check_attention(const hy_paged_cache* cache, const hy_paged_batch* batch, int rows, int q_heads, int dtype)
{
    int rc = check_cache(cache);
    if (!rc) rc = check_batch(batch, cache);
    if (!rc) rc = check_dtype(rows, dtype);
    if (rc) return rc;
    if (q_heads < 1 || q_heads % cache->num_kv_heads)
        return fail(HY_ERR_INVALID_ARGUMENT, "q_heads must be a positive multiple of num_kv_heads");
    if (q_heads > 1024) return fail(HY_ERR_UNSUPPORTED, "q_heads must be at most 1024");
    if (static_cast<long long>(rows) * q_heads > INT_MAX)
        return fail(HY_ERR_CAPACITY, "rows * q_heads must be below 2^31");
    return HY_OK;
}

// Scale, window and sinks of a call.
inline int check_view(float scale, int causal, int window, int sinks)
{
    if (window < 0 || sinks < 0) return fail(HY_ERR_INVALID_ARGUMENT, "window and sinks must not be negative");
    if (!causal && window > 0) return fail(HY_ERR_UNSUPPORTED, "a window needs causal attention");
    const float scale_log2 = scale * 1.4426950408889634f;
    if (!(scale > 0.f) || scale_log2 - scale_log2 != 0.f)
        return fail(HY_ERR_INVALID_ARGUMENT, "scale must be positive, and finite times log2(e) too");
    return HY_OK;
}

// The lse of a call's rows.
inline int check_lse(const float* lse, int rows, int q_heads, long long row_stride, long long head_stride)
{
    if (row_stride < 0 || head_stride < 0) return fail(HY_ERR_INVALID_ARGUMENT, "lse strides must not be negative");
    if (reinterpret_cast<uintptr_t>(lse) % 4 != 0) return fail(HY_ERR_INVALID_ARGUMENT, "lse must be aligned to 4 bytes");
    return check_apart("lse", rows, q_heads, 1, row_stride, head_stride);
}

// Weights of the cache's positions. (A dimension with one entry is not stepped over.)
inline int check_weights(const hy_paged_weights* w, const hy_paged_cache* c)
{
    if (!w || !w->weights_dev) return fail(HY_ERR_INVALID_ARGUMENT, "weights are null");
    if (reinterpret_cast<uintptr_t>(w->weights_dev) % 4 != 0) return fail(HY_ERR_INVALID_ARGUMENT, "weights must be aligned to 4 bytes");
    if (w->page_stride < 0 || w->head_stride < 0 || w->row_stride < 0)
        return fail(HY_ERR_INVALID_ARGUMENT, "weight strides must not be negative");
    if ((c->num_pages > 1 && w->page_stride == 0) || (c->num_kv_heads > 1 && w->head_stride == 0) || (c->page_size > 1 && w->row_stride == 0))
        return fail(HY_ERR_INVALID_ARGUMENT, "weights must not overlap");
    return HY_OK;
}

}  // namespace hy
