// Paged attention of fp32 rows.
#include "hy_paged_launch.cuh"

cudaError_t hy_internal::paged_attention_f32(const hy::PagedAttnArgs& a, int cache_dtype, int head_dim, int cols, int device,
                                             cudaStream_t s)
{
    return hy::launch_split_typed<float>(a, cache_dtype, head_dim, cols, device, s);
}
