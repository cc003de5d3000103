// Launches of the paged attention, one translation unit per row type
// (hy_paged_attn_f32.cu, hy_paged_attn_bf16.cu).
#pragma once

#include <algorithm>
#include <atomic>
#include <cstring>
#include <type_traits>

#include "hy_decode.h"
#include "hy_paged_attn.cuh"
#include "hy_paged_chunk.cuh"
#include "hy_paged.h"

namespace hy_internal {
cudaError_t paged_attention_f32(const hy::PagedAttnArgs& a, int cache_dtype, int head_dim, int cols, int device, cudaStream_t s);
cudaError_t paged_attention_bf16(const hy::PagedAttnArgs& a, int cache_dtype, int head_dim, int cols, int device, cudaStream_t s);
}  // namespace hy_internal

namespace hy {

template <typename T>
struct Tag {
    using type = T;
};

// f(row type, cache type, head_dim) with the run-time types as types.
template <typename RT, typename F>
auto with_types(RT rt, int cache_dtype, int head_dim, F&& f)
{
    auto dim = [&](auto ct) {
        return head_dim == 64 ? f(rt, ct, std::integral_constant<int, 64>{})
                              : f(rt, ct, std::integral_constant<int, 128>{});
    };
    switch (cache_dtype)
    {
    case HY_DTYPE_F32: return dim(Tag<float>{});
    case HY_DTYPE_BF16: return dim(Tag<__nv_bfloat16>{});
    case HY_DTYPE_E4M3: return dim(Tag<E4M3>{});
    default: return dim(Tag<Int8>{});
    }
}
template <typename F>
auto with_row_type(int row_dtype, int cache_dtype, int head_dim, F&& f)
{
    return row_dtype == HY_DTYPE_F32 ? with_types(Tag<float>{}, cache_dtype, head_dim, f)
                                     : with_types(Tag<__nv_bfloat16>{}, cache_dtype, head_dim, f);
}

// Lets Kernel have `smem` bytes of dynamic shared memory; set once per device.
template <auto Kernel>
cudaError_t allow_smem(int smem, int device)
{
    static std::atomic<unsigned long long> done{0};
    const unsigned long long bit = 1ull << (device & 63);
    if (device < 64 && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
    const cudaError_t e =
        cudaFuncSetAttribute(reinterpret_cast<const void*>(Kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && device < 64) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// A launch that may be prepared while the kernel before it in the stream runs (the kernels wait for its end).
template <typename... Args>
cudaError_t launch_pdl(void (*kernel)(Args...), dim3 grid, int threads, int smem, cudaStream_t s, const Args&... args)
{
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename E>
cudaError_t launch_split(const PagedAttnArgs& a, int device, cudaStream_t s)
{
    using Sh = SplitShape<E>;
    cudaError_t e = allow_smem<paged_split_kernel<E>>(Sh::SMEM, device);
    if (e == cudaSuccess) e = launch_pdl(paged_split_kernel<E>, dim3(Sh::GRID), kSplitThreads, Sh::SMEM, s, a);
    if (e == cudaSuccess)
        e = launch_pdl(paged_join_kernel<E>, dim3(Sh::GRID, (E::COLS + 7) / 8), kJoinThreads, 0, s, a);
    return e;
}

// Tensor maps of K and V for blocks fetched 16 rows of a page at a time. Pages that do not
// hold a multiple of 16 rows, and layouts that the maps cannot express, are copied row by row.
template <typename CT, int D>
ChunkTma chunk_tma(const PagedAttnArgs& a)
{
    using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const EncodeFn encode = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            fn = nullptr;
        return reinterpret_cast<EncodeFn>(fn);
    }();
    ChunkTma t;
    std::memset(&t, 0, sizeof t);
    if (!encode || a.c.page_size % 16 != 0) return t;
    constexpr int E = sizeof(CT);
    struct Dim {
        long long stride;
        cuuint64_t size;
        cuuint32_t box;
        int* where;
    } dims[3] = {{a.c.row_stride, static_cast<cuuint64_t>(a.c.page_size), 16, &t.row_c},
                 {a.c.head_stride, static_cast<cuuint64_t>(a.c.kv_heads), 1, &t.head_c},
                 {a.c.page_stride, static_cast<cuuint64_t>(a.c.num_pages), 1, &t.page_c}};
    std::sort(dims, dims + 3, [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
    const cuuint32_t inner = E == 1 ? D : 64;   // 128 bytes of a bf16 row, a row of codes
    cuuint64_t size[4] = {D}, stride[3];
    cuuint32_t box[4] = {inner}, step[4] = {1, 1, 1, 1};
    for (int i = 0; i < 3; ++i)
    {
        if (dims[i].stride <= 0 || dims[i].stride * E >= (1ll << 40)) return t;
        size[i + 1] = dims[i].size;
        stride[i] = static_cast<cuuint64_t>(dims[i].stride) * E;
        box[i + 1] = dims[i].box;
        *dims[i].where = i + 1;
    }
    for (int v = 0; v < 2; ++v)
        if (encode(v ? &t.v : &t.k, E == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, v ? a.c.v : a.c.k,
                   size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   E == 1 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return t;
    t.on = 1;
    return t;
}

template <typename CT, int D>
cudaError_t launch_chunk(const PagedAttnArgs& a, int device, cudaStream_t s)
{
    using E = ChunkEngine<CT, D>;
    const ChunkTma tma = chunk_tma<CT, D>(a);
    cudaError_t e = allow_smem<paged_chunk_kernel<CT, D>>(E::SMEM, device);
    if (e == cudaSuccess) e = launch_pdl(paged_chunk_kernel<CT, D>, dim3(148), kChunkThreads, E::SMEM, s, a, tma);
    if (e == cudaSuccess) e = launch_pdl(paged_join_wide_kernel<E>, dim3(148, 8), kJoinThreads, 0, s, a);
    return e;
}

template <typename QT>
cudaError_t launch_split_typed(const PagedAttnArgs& a, int cache_dtype, int head_dim, int cols, int device, cudaStream_t s)
{
    return with_types(Tag<QT>{}, cache_dtype, head_dim, [&](auto, auto ct, auto d) {
        using CT = typename decltype(ct)::type;
        constexpr int D = decltype(d)::value;
        if constexpr (std::is_same_v<CT, float>)
        {
            if (cols == 2) return launch_split<FmaEngine<QT, D, 2>>(a, device, s);
            if (cols == 4) return launch_split<FmaEngine<QT, D, 4>>(a, device, s);
        }
        if constexpr (std::is_same_v<QT, __nv_bfloat16> && !std::is_same_v<CT, float>)
            if (cols == 256) return launch_chunk<CT, D>(a, device, s);
        return cols <= 8    ? launch_split<MmaEngine<QT, CT, D, 1>>(a, device, s)
               : cols == 16 ? launch_split<MmaEngine<QT, CT, D, 2>>(a, device, s)
                            : launch_split<MmaEngine<QT, CT, D, 4>>(a, device, s);
    });
}

}  // namespace hy
