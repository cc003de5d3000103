// C ABI of the paged KV cache (include/hy_paged.h): checks of arguments, the
// choice of kernels, launches. Every check that needs no device comes before
// the first CUDA call.
#include <algorithm>

#include "hy_call.cuh"
#include "hy_paged_launch.cuh"

using namespace hy;

namespace {

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
    return hy_paged_attention_lse(cache, batch, rows, q_heads, dtype, q_dev, q_row_stride, q_head_stride, out_dev,
                                  out_row_stride, out_head_stride, nullptr, 0, 0, scale, causal, window, sinks,
                                  workspace_dev, workspace_bytes, stream);
}

int hy_paged_attention_lse(const hy_paged_cache* cache, const hy_paged_batch* batch, int rows, int q_heads, int dtype,
                           const void* q_dev, int64_t q_row_stride, int64_t q_head_stride, void* out_dev,
                           int64_t out_row_stride, int64_t out_head_stride, float* lse_dev, int64_t lse_row_stride,
                           int64_t lse_head_stride, float scale, int causal, int window, int sinks,
                           void* workspace_dev, size_t workspace_bytes, void* stream)
{
    int rc = check_attention(cache, batch, rows, q_heads, dtype);
    if (rc) return rc;
    rc = check_view(scale, causal, window, sinks);
    if (rc) return rc;
    if (rows == 0 || batch->num_seqs == 0) return HY_OK;
    rc = check_rows("q", q_dev, rows, q_heads, q_row_stride, q_head_stride, dtype);
    if (!rc) rc = check_rows("out", out_dev, rows, q_heads, out_row_stride, out_head_stride, dtype);
    if (!rc) rc = check_apart("out", rows, q_heads, cache->head_dim, out_row_stride, out_head_stride);
    if (rc) return rc;
    if (q_dev == out_dev) return fail(HY_ERR_INVALID_ARGUMENT, "q and out must not overlap");
    if (lse_dev)
    {
        rc = check_lse(lse_dev, rows, q_heads, lse_row_stride, lse_head_stride);
        if (rc) return rc;
        if (lse_dev == out_dev || lse_dev == q_dev) return fail(HY_ERR_INVALID_ARGUMENT, "lse must not overlap q or out");
    }
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
                          power_of_two(cache->page_size), power_of_two(group), scale * 1.4426950408889634f, workspace_dev,
                          lse_dev, lse_row_stride, lse_head_stride};
    const int cols = tile_columns(batch->max_rows, group, dtype, cache->dtype);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const auto launch = dtype == HY_DTYPE_F32 ? hy_internal::paged_attention_f32 : hy_internal::paged_attention_bf16;
    const cudaError_t e = launch(a, cache->dtype, cache->head_dim, cols, cache->device, s);
    return e == cudaSuccess ? HY_OK : cuda_fail("paged attention", e);
}

}  // extern "C"
