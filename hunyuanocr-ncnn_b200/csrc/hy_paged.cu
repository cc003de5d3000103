// C ABI of the paged KV cache (include/hy_paged.h): checks of arguments, the
// choice of kernels, launches. Every check that needs no device comes before
// the first CUDA call.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <string>

#include "hy_paged.cuh"
#include "hy_paged_launch.cuh"
#include "hy_paged.h"

namespace hy_internal {
void set_last_error(const std::string& msg);
}  // namespace hy_internal

using namespace hy;

namespace {

int fail(int code, const char* msg) noexcept
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

int cuda_fail(const char* what, cudaError_t e) noexcept
{
    char msg[256];
    snprintf(msg, sizeof msg, "%s: %s", what, cudaGetErrorString(e));
    return fail(e == cudaErrorMemoryAllocation ? HY_ERR_OUT_OF_MEMORY : HY_ERR_CUDA, msg);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// log2 of n where it is one, else -1.
int power_of_two(int n)
{
    if (n & (n - 1)) return -1;
    int s = 0;
    while ((1 << s) < n) ++s;
    return s;
}

// A stride of a dimension with one entry is never taken.
bool off16(long long stride, int elem, int entries) { return entries > 1 && stride * elem % 16 != 0; }

int elem_size(int dtype) { return dtype == HY_DTYPE_F32 ? 4 : dtype == HY_DTYPE_BF16 ? 2 : 1; }

int check_cache(const hy_paged_cache* c)
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

int check_batch(const hy_paged_batch* b, const hy_paged_cache* c)
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

int check_rows(const char* name, const void* p, int rows, int heads, long long row_stride, long long head_stride, int dtype)
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
int check_apart(const char* name, int rows, int heads, int head_dim, long long row_stride, long long head_stride)
{
    if ((rows < 2 || row_stride >= head_dim) && (heads < 2 || head_stride >= head_dim)) return HY_OK;
    char msg[96];
    snprintf(msg, sizeof msg, "%s rows must not overlap", name);
    return fail(HY_ERR_INVALID_ARGUMENT, msg);
}

int check_dtype(int rows, int dtype)
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

PagedCache device_cache(const hy_paged_cache* c)
{
    return {c->k_dev, c->v_dev, c->k_scale_dev, c->v_scale_dev, c->page_stride, c->head_stride, c->row_stride,
            c->scale_page_stride, c->scale_head_stride, c->scale_row_stride, c->num_pages, c->page_size,
            c->num_kv_heads, c->status_dev};
}

PagedBatch device_batch(const hy_paged_batch* b, int rows)
{
    return {b->q_start_dev, b->kv_len_dev, b->block_table_dev, b->table_stride, b->table_width, b->num_seqs, rows};
}

int paged_rows(bool write, const hy_paged_cache* cache, const hy_paged_batch* batch, int rows, int dtype, void* k,
               long long krs, long long khs, void* v, long long vrs, long long vhs, void* stream)
{
    int rc = check_cache(cache);
    if (!rc) rc = check_batch(batch, cache);
    if (!rc) rc = check_dtype(rows, dtype);
    if (rc) return rc;
    if (rows == 0 || batch->num_seqs == 0) return HY_OK;
    rc = check_rows("k", k, rows, cache->num_kv_heads, krs, khs, dtype);
    if (!rc) rc = check_rows("v", v, rows, cache->num_kv_heads, vrs, vhs, dtype);
    if (!rc && !write) rc = check_apart("k", rows, cache->num_kv_heads, cache->head_dim, krs, khs);
    if (!rc && !write) rc = check_apart("v", rows, cache->num_kv_heads, cache->head_dim, vrs, vhs);
    if (rc) return rc;
    if (!write && k == v) return fail(HY_ERR_INVALID_ARGUMENT, "k and v must not overlap");
    for (const long long x : {krs, khs, vrs, vhs, static_cast<long long>(cache->head_stride), static_cast<long long>(cache->scale_head_stride)})
        if (x > INT_MAX) return fail(HY_ERR_CAPACITY, "row and head strides must be below 2^31");
    DeviceGuard guard(cache->device);
    if (guard.error() != cudaSuccess) return cuda_fail("device", guard.error());
    PagedRowArgs a{device_cache(cache), device_batch(batch, rows), k, v, static_cast<int>(krs), static_cast<int>(khs),
                   static_cast<int>(vrs), static_cast<int>(vhs), static_cast<int>(cache->head_stride),
                   static_cast<int>(cache->scale_head_stride), 1, 0};
    // Rows of a CTA: one while that leaves the GPU fewer than 8 CTAs per SM, then more; at most 2^16 vectors.
    a.per_cta = std::min({kRowsPerCta, std::max(1, rows / (8 * 148)), std::max(1, 32768 / cache->num_kv_heads - 1)});
    a.vectors_inv = static_cast<unsigned>(((1ull << 32) + 2u * cache->num_kv_heads - 1) / (2u * cache->num_kv_heads));
    const cudaError_t e = with_row_type(dtype, cache->dtype, cache->head_dim, [&](auto rt, auto ct, auto d) {
        using RT = typename decltype(rt)::type;
        using CT = typename decltype(ct)::type;
        constexpr int D = decltype(d)::value;
        return launch_pdl(write ? paged_write_kernel<RT, CT, D> : paged_read_kernel<RT, CT, D>,
                          dim3((rows + a.per_cta - 1) / a.per_cta), kRowWarps * 32, 0, static_cast<cudaStream_t>(stream), a);
    });
    return e == cudaSuccess ? HY_OK : cuda_fail(write ? "paged write" : "paged read", e);
}

// Columns of a tile: as many as a sequence's rows need, up to 32, in the split
// kernels (fp32 caches have tiles of 2 and 4 too, FmaEngine), else 256, for which
// bf16 rows take the tcgen05 kernel; fp32 rows and fp32 caches stay at 32.
// The border, in us with tiles of 32 / 256 columns (16 sequences at 8192 keys, 8 KV heads
// of 128): 24 columns 114 / 134, 32 columns 117 / 135, 40 columns 201 / 135 (bf16 cache);
// 32 columns 152 / 221, 40 columns 269 / 222 (INT8); one sequence at 2048 keys: 32 columns
// 17.8 / 18.6, 40 columns 18.9 / 18.8 (bf16), 18.1 / 22.5 and 19.9 / 23.1 (INT8): the wide kernel pays where
// there are many sequences or long ones. The choice is the call's: 63 tokens and a chunk of 512 rows at 1024-8192
// E4M3 keys take 581 us in one call, 106 and 91 us in two.
int tile_columns(int max_rows, int group, int dtype, int cache_dtype)
{
    const long long cols = static_cast<long long>(max_rows) * group;
    if (cache_dtype == HY_DTYPE_F32 && cols <= 4) return cols <= 2 ? 2 : 4;
    if (cols > 32 && dtype == HY_DTYPE_BF16 && cache_dtype != HY_DTYPE_F32) return 256;
    return cols <= 8 ? 8 : cols <= 16 ? 16 : 32;
}

int check_attention(const hy_paged_cache* cache, const hy_paged_batch* batch, int rows, int q_heads, int dtype)
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

// Descriptions and two parts for every CTA.
size_t attention_workspace(const hy_paged_cache* cache, const hy_paged_batch* batch, int q_heads, int dtype)
{
    const int cols = tile_columns(batch->max_rows, q_heads / cache->num_kv_heads, dtype, cache->dtype);
    return kSplitDescBytes + static_cast<size_t>(2 * (cols == 256 ? 148 : kSplitMaxCtas)) * cols * (cache->head_dim + 2) * sizeof(float);
}

}  // namespace

extern "C" {

int hy_paged_kv_write(const hy_paged_cache* cache, const hy_paged_batch* batch, int rows, int dtype, const void* k_dev,
                      int64_t k_row_stride, int64_t k_head_stride, const void* v_dev, int64_t v_row_stride,
                      int64_t v_head_stride, void* stream)
{
    return paged_rows(true, cache, batch, rows, dtype, const_cast<void*>(k_dev), k_row_stride, k_head_stride,
                      const_cast<void*>(v_dev), v_row_stride, v_head_stride, stream);
}

int hy_paged_kv_read(const hy_paged_cache* cache, const hy_paged_batch* batch, int rows, int dtype, void* k_dev,
                     int64_t k_row_stride, int64_t k_head_stride, void* v_dev, int64_t v_row_stride,
                     int64_t v_head_stride, void* stream)
{
    return paged_rows(false, cache, batch, rows, dtype, k_dev, k_row_stride, k_head_stride, v_dev, v_row_stride,
                      v_head_stride, stream);
}

int hy_paged_attention_workspace(const hy_paged_cache* cache, const hy_paged_batch* batch, int rows, int q_heads,
                                 int dtype, size_t* bytes)
{
    const int rc = check_attention(cache, batch, rows, q_heads, dtype);
    if (rc) return rc;
    if (!bytes) return fail(HY_ERR_INVALID_ARGUMENT, "bytes is null");
    *bytes = attention_workspace(cache, batch, q_heads, dtype);
    return HY_OK;
}

int hy_paged_attention(const hy_paged_cache* cache, const hy_paged_batch* batch, int rows, int q_heads, int dtype,
                       const void* q_dev, int64_t q_row_stride, int64_t q_head_stride, void* out_dev,
                       int64_t out_row_stride, int64_t out_head_stride, float scale, int causal, int window, int sinks,
                       void* workspace_dev, size_t workspace_bytes, void* stream)
{
    int rc = check_attention(cache, batch, rows, q_heads, dtype);
    if (rc) return rc;
    if (window < 0 || sinks < 0) return fail(HY_ERR_INVALID_ARGUMENT, "window and sinks must not be negative");
    if (!causal && window > 0) return fail(HY_ERR_UNSUPPORTED, "a window needs causal attention");
    const float scale_log2 = scale * 1.4426950408889634f;
    if (!(scale > 0.f) || scale_log2 - scale_log2 != 0.f)
        return fail(HY_ERR_INVALID_ARGUMENT, "scale must be positive, and finite times log2(e) too");
    if (rows == 0 || batch->num_seqs == 0) return HY_OK;
    rc = check_rows("q", q_dev, rows, q_heads, q_row_stride, q_head_stride, dtype);
    if (!rc) rc = check_rows("out", out_dev, rows, q_heads, out_row_stride, out_head_stride, dtype);
    if (!rc) rc = check_apart("out", rows, q_heads, cache->head_dim, out_row_stride, out_head_stride);
    if (rc) return rc;
    if (q_dev == out_dev) return fail(HY_ERR_INVALID_ARGUMENT, "q and out must not overlap");
    if (!workspace_dev || !aligned16(workspace_dev))
        return fail(HY_ERR_INVALID_ARGUMENT, "the workspace is null or not on 16 bytes");
    if (workspace_bytes < attention_workspace(cache, batch, q_heads, dtype))
        return fail(HY_ERR_CAPACITY, "the workspace is too small");
    DeviceGuard guard(cache->device);
    if (guard.error() != cudaSuccess) return cuda_fail("device", guard.error());
    const int group = q_heads / cache->num_kv_heads;
    // Positions lie below 2^30: wider windows and more sinks change nothing, and sums with these stay within 32 bits.
    window = std::min(window, 1 << 30);
    sinks = std::min(sinks, 1 << 30);
    const PagedAttnArgs a{device_cache(cache), device_batch(batch, rows), q_dev, out_dev, q_row_stride, q_head_stride,
                          out_row_stride, out_head_stride, q_heads, group, causal != 0, window, window > 0 ? sinks : 0,
                          power_of_two(cache->page_size), power_of_two(group), scale_log2, workspace_dev};
    const int cols = tile_columns(batch->max_rows, group, dtype, cache->dtype);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const auto launch = dtype == HY_DTYPE_F32 ? hy_internal::paged_attention_f32 : hy_internal::paged_attention_bf16;
    const cudaError_t e = launch(a, cache->dtype, cache->head_dim, cols, cache->device, s);
    return e == cudaSuccess ? HY_OK : cuda_fail("paged attention", e);
}

}  // extern "C"
