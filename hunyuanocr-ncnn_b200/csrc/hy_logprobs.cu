// C ABI of the log probabilities (include/hy_logprobs.h): checks of arguments, launches.
#include <algorithm>

#include "hy_call.cuh"
#include "hy_logprobs.cuh"
#include "hy_logprobs.h"
#include "hy_paged_launch.cuh"

using namespace hy;

namespace {

template <typename T, bool TOP, int THREADS>
cudaError_t launch_logprobs(const LogprobArgs& a, int device, cudaStream_t s)
{
    const int smem = TOP ? (a.iters + kLogprobRun - 1) / kLogprobRun * THREADS * static_cast<int>(sizeof(float)) : 0;
    cudaError_t e = allow_smem<logprob_kernel<T, TOP, THREADS>>(16 * 1024, device);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.rows * a.split);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, logprob_kernel<T, TOP, THREADS>, a);
}

template <typename T>
cudaError_t launch_logprobs(LogprobArgs a, int device, cudaStream_t s)
{
    // CTAs of a row: more while the rows leave SMs without work, of at least 4096 logits each (1024 rows of 120818: 75 us
    // with one, 85 with four; 200 rows 27 and 19).
    while (a.split < kLogprobMaxCluster && ((a.rows * a.split < 4 * 148 && a.vocab / a.split > 4096) || a.vocab / a.split > (1 << 18))) a.split *= 2;
    constexpr int EV = 16 / static_cast<int>(sizeof(T));
    const bool few = a.rows * a.split < 148;
    const int vectors = (a.vocab + 2 * EV - 2) / EV;   // (a row may start anywhere in its first vector)
    const int step = (few ? kLogprobFewThreads : kLogprobManyThreads) * (32 / EV);
    a.iters = (vectors + a.split * step - 1) / (a.split * step);
    if (few)
        return a.top ? launch_logprobs<T, true, kLogprobFewThreads>(a, device, s) : launch_logprobs<T, false, kLogprobFewThreads>(a, device, s);
    return a.top ? launch_logprobs<T, true, kLogprobManyThreads>(a, device, s) : launch_logprobs<T, false, kLogprobManyThreads>(a, device, s);
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
    // (the kernel's index of a token, a step of threads ahead of the last, stays within 32 bits)
    if (tokens_per_row > 1 << 30) return fail(HY_ERR_CAPACITY, "tokens_per_row must be at most 2^30");
    if (rows == 0) return HY_OK;
    if (!logits_dev || (tokens_per_row > 0 && (!tokens_dev || !logprobs_dev)) || (top > 0 && (!top_ids_dev || !top_logprobs_dev)))
        return fail(HY_ERR_INVALID_ARGUMENT, "logits, tokens or an output is null");
    if (reinterpret_cast<uintptr_t>(logits_dev) % elem_size(dtype) != 0)
        return fail(HY_ERR_INVALID_ARGUMENT, "logits must be aligned to their type");
    DeviceGuard guard(device);
    if (guard.error() != cudaSuccess) return cuda_fail("device", guard.error());
    LogprobArgs a{logits_dev, row_stride, rows, vocab, tokens_dev, tokens_per_row, top, logprobs_dev, entropy_dev,
                  top_ids_dev, top_logprobs_dev, 1, 1};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == HY_DTYPE_F32 ? launch_logprobs<float>(a, device, s) : launch_logprobs<__nv_bfloat16>(a, device, s);
    return e == cudaSuccess ? HY_OK : cuda_fail("log probabilities", e);
}

}  // extern "C"
