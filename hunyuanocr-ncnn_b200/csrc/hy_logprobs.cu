// C ABI of the log probabilities (include/hy_logprobs.h): checks of arguments, launches.
#include <algorithm>

#include "hy_call.cuh"
#include "hy_logprobs.cuh"
#include "hy_logprobs.h"
#include "hy_paged_launch.cuh"

using namespace hy;

namespace {

template <typename T, bool TOP>
cudaError_t launch_logprobs(const LogprobArgs& a, int device, cudaStream_t s)
{
    const int smem = TOP ? a.iters * kLogprobThreads * static_cast<int>(sizeof(float)) : 0;
    cudaError_t e = allow_smem<logprob_kernel<T, TOP>>(160 * 1024, device);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.rows * a.split);
    cfg.blockDim = dim3(kLogprobThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, logprob_kernel<T, TOP>, a);
}

}  // namespace

extern "C" {

int hy_token_logprobs(const void* logits_dev, int rows, int vocab, int64_t row_stride, int dtype, int device,
                      const int* tokens_dev, int tokens_per_row, int top, float* logprobs_dev, float* entropy_dev,
                      int* top_ids_dev, float* top_logprobs_dev, void* stream)
{
    int rc = check_dtype(rows, dtype);
    if (rc) return rc;
    if (vocab < 1 || vocab > (1 << 20)) return fail(HY_ERR_INVALID_ARGUMENT, "vocab must be in 1..2^20");
    if (tokens_per_row < 0) return fail(HY_ERR_INVALID_ARGUMENT, "tokens_per_row must not be negative");
    if (top < 0 || top > HY_LOGPROBS_MAX_TOP || top > vocab)
        return fail(HY_ERR_INVALID_ARGUMENT, "top must be in 0..64 and at most vocab");
    if (row_stride < 0) return fail(HY_ERR_INVALID_ARGUMENT, "row_stride must not be negative");
    if (device < 0) return fail(HY_ERR_INVALID_ARGUMENT, "device must not be negative");
    if (static_cast<long long>(rows) * std::max({tokens_per_row, top, kLogprobMaxCluster}) > INT_MAX)
        return fail(HY_ERR_CAPACITY, "rows * max(tokens_per_row, top, 8) must be below 2^31");
    if (rows == 0) return HY_OK;
    if (!logits_dev || (tokens_per_row > 0 && (!tokens_dev || !logprobs_dev)) || (top > 0 && (!top_ids_dev || !top_logprobs_dev)))
        return fail(HY_ERR_INVALID_ARGUMENT, "logits, tokens or an output is null");
    if (reinterpret_cast<uintptr_t>(logits_dev) % elem_size(dtype) != 0)
        return fail(HY_ERR_INVALID_ARGUMENT, "logits must be aligned to their type");
    DeviceGuard guard(device);
    if (guard.error() != cudaSuccess) return cuda_fail("device", guard.error());
    LogprobArgs a{logits_dev, row_stride, rows, vocab, tokens_dev, tokens_per_row, top, logprobs_dev, entropy_dev,
                  top_ids_dev, top_logprobs_dev, 1, 1};
    // CTAs of a row: more while the rows leave SMs without one, of at least 4096 logits each.
    while (a.split < kLogprobMaxCluster && ((rows * a.split < 4 * 148 && vocab / a.split > 4096) || vocab / a.split > (1 << 18))) a.split *= 2;
    const int ev = 16 / elem_size(dtype), vectors = (vocab + 2 * ev - 2) / ev;   // (a row may start anywhere in its first vector)
    const int step = kLogprobThreads * (32 / ev);
    a.iters = (vectors + a.split * step - 1) / (a.split * step);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (dtype == HY_DTYPE_F32) e = top ? launch_logprobs<float, true>(a, device, s) : launch_logprobs<float, false>(a, device, s);
    else e = top ? launch_logprobs<__nv_bfloat16, true>(a, device, s) : launch_logprobs<__nv_bfloat16, false>(a, device, s);
    return e == cudaSuccess ? HY_OK : cuda_fail("log probabilities", e);
}

}  // extern "C"
