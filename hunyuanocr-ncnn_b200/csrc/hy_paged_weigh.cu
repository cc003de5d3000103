// C ABI of the attention weights of cached positions and of the eviction by them
// (hy_paged_add_weights and hy_paged_evict of include/hy_paged.h): checks of
// arguments, the choice of kernels, launches.
#include <algorithm>

#include "hy_call.cuh"
#include "hy_paged_evict.cuh"
#include "hy_paged_launch.cuh"
#include "hy_paged_weigh.cuh"
#include "hy_paged_weigh_chunk.cuh"

using namespace hy;

namespace {

template <typename E>
cudaError_t launch_weigh(const PagedWeighArgs& w, int device, cudaStream_t s)
{
    const cudaError_t e = allow_smem<paged_weigh_kernel<E>>(WeighShape<E>::SMEM, device);
    return e != cudaSuccess ? e : launch_pdl(paged_weigh_kernel<E>, dim3(148 * kWeighCtas), kSplitThreads, WeighShape<E>::SMEM, s, w);
}

template <typename QT, typename CT, int D>
cudaError_t launch_weigh_wide(const PagedWeighArgs& w, int device, cudaStream_t s)
{
    using E = WeighWide<QT, CT, D>;
    const cudaError_t e = allow_smem<paged_weigh_wide_kernel<E>>(E::SMEM, device);
    return e != cudaSuccess ? e : launch_pdl(paged_weigh_wide_kernel<E>, dim3(148), kWeighWideWarps * 32, E::SMEM, s, w);
}

// Tensor map of q, whose boxes are tiles of 128 columns: groups that divide 128, and rows a whole number of heads apart.
template <int D>
WeighTma weigh_tma(const PagedAttnArgs& a)
{
    WeighTma t;
    std::memset(&t, 0, sizeof t);
    const auto encode = tensor_map_encoder();
    const long long head = (a.q_heads > 1 ? a.q_head_stride : D) * 2, row = a.b.rows > 1 ? a.q_row_stride * 2 : head * a.q_heads;
    if (!encode || 128 % a.group != 0 || head < 16 || row < head || row % head != 0 || row >= (1ll << 40)) return t;
    const cuuint64_t size[3] = {D, static_cast<cuuint64_t>(a.q_heads), static_cast<cuuint64_t>(a.b.rows)};
    const cuuint64_t stride[2] = {static_cast<cuuint64_t>(head), static_cast<cuuint64_t>(row)};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(a.group), static_cast<cuuint32_t>(128 / a.group)}, step[3] = {1, 1, 1};
    t.on = encode(&t.q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(a.q), size, stride, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    return t;
}

template <typename CT, int D>
cudaError_t launch_weigh_chunk(const PagedWeighArgs& w, int device, cudaStream_t s)
{
    using E = WeighChunk<CT, D>;
    const WeighTma tma = weigh_tma<D>(w.a);
    const cudaError_t e = allow_smem<paged_weigh_chunk_kernel<CT, D>>(E::SMEM, device);
    return e != cudaSuccess ? e : launch_pdl(paged_weigh_chunk_kernel<CT, D>, dim3(148), kWeighChunkThreads, E::SMEM, s, w, tma);
}

}  // namespace

extern "C" {

int hy_paged_add_weights(const hy_paged_cache* cache, const hy_paged_batch* batch, int rows, int q_heads, int dtype,
                         const void* q_dev, int64_t q_row_stride, int64_t q_head_stride, const float* lse_dev,
                         int64_t lse_row_stride, int64_t lse_head_stride, float scale, int causal, int window,
                         int sinks, const hy_paged_weights* weights, void* stream)
{
    int rc = check_attention(cache, batch, rows, q_heads, dtype);
    if (!rc) rc = check_view(scale, causal, window, sinks);
    if (!rc) rc = check_weights(weights, cache);
    if (rc) return rc;
    if (static_cast<long long>(rows) * q_heads >= kWeighAll) return fail(HY_ERR_CAPACITY, "rows * q_heads must be below 2^30");
    if (rows == 0 || batch->num_seqs == 0) return HY_OK;
    rc = check_rows("q", q_dev, rows, q_heads, q_row_stride, q_head_stride, dtype);
    if (!rc && !lse_dev) rc = fail(HY_ERR_INVALID_ARGUMENT, "lse is null");
    if (!rc) rc = check_lse(lse_dev, rows, q_heads, lse_row_stride, lse_head_stride);
    if (rc) return rc;
    if (weights->weights_dev == lse_dev) return fail(HY_ERR_INVALID_ARGUMENT, "weights and lse must not overlap");
    DeviceGuard guard(cache->device);
    if (guard.error() != cudaSuccess) return cuda_fail("device", guard.error());
    const int group = q_heads / cache->num_kv_heads;
    // Positions lie below 2^30: wider windows and more sinks change nothing, and sums with these stay within 32 bits.
    window = std::min(window, 1 << 30);
    sinks = std::min(sinks, 1 << 30);
    PagedWeighArgs w{};
    w.a = {device_cache(cache), device_batch(batch, rows), q_dev, nullptr, q_row_stride, q_head_stride, 0, 0, q_heads, group,
           causal != 0, window, window > 0 ? sinks : 0, power_of_two(cache->page_size), power_of_two(group), 0.f, nullptr,
           const_cast<float*>(lse_dev), lse_row_stride, lse_head_stride};
    w.weights = weights->weights_dev;
    w.w_page_stride = weights->page_stride;
    w.w_head_stride = weights->head_stride;
    w.w_row_stride = weights->row_stride;
    w.scale = scale;
    const long long cols = static_cast<long long>(batch->max_rows) * group;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = with_row_type(dtype, cache->dtype, cache->head_dim, [&](auto rt, auto ct, auto d) {
        using RT = typename decltype(rt)::type;
        using CT = typename decltype(ct)::type;
        constexpr int D = decltype(d)::value;
        if constexpr (std::is_same_v<CT, float>)
        {
            if (cols <= 2) return launch_weigh<WeighFma<RT, D, 2>>(w, cache->device, s);
            if (cols <= 4) return launch_weigh<WeighFma<RT, D, 4>>(w, cache->device, s);
        }
        else if (cols <= 8) return launch_weigh<WeighMma<RT, CT, D>>(w, cache->device, s);
        if constexpr (std::is_same_v<RT, __nv_bfloat16> && !std::is_same_v<CT, float>)
            if (cols > 32) return launch_weigh_chunk<CT, D>(w, cache->device, s);
        return launch_weigh_wide<RT, CT, D>(w, cache->device, s);
    });
    return e == cudaSuccess ? HY_OK : cuda_fail("attention weights", e);
}

int hy_paged_evict(const hy_paged_cache* cache, const hy_paged_batch* batch, int keep, int first, int recent,
                   const hy_paged_weights* weights, int* kv_len_dev, int* kept_dev, void* stream)
{
    int rc = check_cache(cache);
    if (!rc) rc = check_batch(batch, cache);
    if (!rc) rc = check_weights(weights, cache);
    if (rc) return rc;
    if (keep < 1 || first < 0 || recent < 0 || static_cast<long long>(first) + recent > keep)
        return fail(HY_ERR_INVALID_ARGUMENT, "keep must be positive, first and recent not negative and together at most keep");
    // (positions lie below 2^30; the kernel's index over the list, a step of threads ahead of it, stays within 32 bits)
    if (keep > 1 << 30) return fail(HY_ERR_INVALID_ARGUMENT, "keep must be at most 2^30");
    if (static_cast<long long>(batch->num_seqs) * cache->num_kv_heads * kEvictMaxCluster > INT_MAX)
        return fail(HY_ERR_CAPACITY, "num_seqs * num_kv_heads must be below 2^28");
    const int e = elem_size(cache->dtype);
    if ((cache->num_pages > 1 && cache->page_stride == 0) || (cache->num_kv_heads > 1 && cache->head_stride == 0) ||
        (cache->page_size > 1 && cache->row_stride == 0) ||
        (e == 1 && ((cache->num_pages > 1 && cache->scale_page_stride == 0) || (cache->num_kv_heads > 1 && cache->scale_head_stride == 0) ||
                    (cache->page_size > 1 && cache->scale_row_stride == 0))))
        return fail(HY_ERR_INVALID_ARGUMENT, "the cache's rows and scales must not overlap");
    if (batch->num_seqs == 0) return HY_OK;
    if (!kept_dev) return fail(HY_ERR_INVALID_ARGUMENT, "kept is null");
    if (kept_dev == batch->kv_len_dev) return fail(HY_ERR_INVALID_ARGUMENT, "kv_len and kept must not overlap");
    if (kv_len_dev && kv_len_dev != batch->kv_len_dev) return fail(HY_ERR_INVALID_ARGUMENT, "kv_len must be the batch's own array");
    DeviceGuard guard(cache->device);
    if (guard.error() != cudaSuccess) return cuda_fail("device", guard.error());
    PagedEvictArgs a{};
    a.c = device_cache(cache);
    a.b = device_batch(batch, 0);
    a.weights = weights->weights_dev;
    a.w_page_stride = weights->page_stride;
    a.w_head_stride = weights->head_stride;
    a.w_row_stride = weights->row_stride;
    a.kept = kept_dev;
    a.kv_len = kv_len_dev;
    a.keep = keep;
    a.first = first;
    a.recent = recent;
    a.elem = e;
    a.pieces = cache->head_dim * e / 16;
    a.page_shift = power_of_two(cache->page_size);
    a.cluster = 1;
    // (84 heads of up to 12579 positions: 140 us with what is behind the first 8192 read again in every step.)
    a.more = static_cast<int>(std::clamp<long long>(static_cast<long long>(batch->table_width) * cache->page_size - kEvictThreads * kEvictHeld, 0, kEvictMore));
    // CTAs of a (sequence, head): more while there are fewer than the GPU holds (two per SM), of one piece a row at least.
    const int items = batch->num_seqs * cache->num_kv_heads;
    while (a.cluster < kEvictMaxCluster && items * a.cluster < 148 && a.cluster < 2 * a.pieces) a.cluster *= 2;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(items * a.cluster);
    cfg.blockDim = dim3(kEvictThreads);
    cfg.dynamicSmemBytes = a.more * sizeof(uint32_t);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaError_t err = allow_smem<paged_evict_kernel>(kEvictMore * sizeof(uint32_t), cache->device);
    if (err == cudaSuccess) err = cudaLaunchKernelEx(&cfg, paged_evict_kernel, a);
    if (err == cudaSuccess && kv_len_dev) err = launch_pdl(evict_lengths_kernel, dim3((batch->num_seqs + 255) / 256), 256, 0, cfg.stream, a);
    return err == cudaSuccess ? HY_OK : cuda_fail("eviction", err);
}

}  // extern "C"
