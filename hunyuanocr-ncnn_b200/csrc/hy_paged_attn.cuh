// Attention of a batch's rows over the paged cache.
//
// out = softmax(scale * q k^T) v over the positions that a row sees, in one
// pass over the keys: a running maximum m, the sum l of exp(s - m) and the sum
// of exp(s - m) v are kept in fp32 and rescaled when m grows.
#pragma once

#include "hy_paged.cuh"

namespace hy {

struct PagedAttnArgs {
    PagedCache c;
    PagedBatch b;
    const void* q;
    void* out;
    long long q_row_stride, q_head_stride, o_row_stride, o_head_stride;
    int q_heads, group;   // group = q_heads / kv_heads
    int causal, window, sinks;
    float scale_log2;     // scale * log2(e)
};

// One warp per (row, query head): right for every case, with no reuse of a key
// between the heads of a group or the rows of a sequence.
template <typename QT, typename CT, int D>
__global__ void __launch_bounds__(128) paged_attn_rows_kernel(const PagedAttnArgs a)
{
    constexpr int E = 4, LPV = D / E, VPW = 32 / LPV;   // keys per step
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long item = static_cast<long long>(blockIdx.x) * 4 + warp;
    if (item >= static_cast<long long>(a.b.rows) * a.q_heads) return;
    const int r = static_cast<int>(item / a.q_heads), h = static_cast<int>(item % a.q_heads), g = h / a.group;
    const int sub = lane / LPV, d = (lane % LPV) * E;
    const int s = paged_find_seq(a.b, r, lane);
    PagedSeq sq;
    if (s < 0 || !paged_seq(a.b, s, a.c.page_size, a.c.status, sq) || r < sq.row0 || r >= sq.row0 + sq.n) return;
    const int p = sq.kv - sq.n + (r - sq.row0);
    const int hi = p < 0 ? 0 : a.causal ? p + 1 : sq.kv;
    const int lo = (a.window > 0) ? max(0, p - a.window + 1) : 0;
    const int ns = min(lo, a.sinks);   // sinks before the window
    const int n = ns + max(0, hi - lo);
    float q[E], acc[E] = {};
    load_row<QT, E>(a.q, r * a.q_row_stride + h * a.q_head_stride + d, q);
    float m = -INFINITY, l = 0.f;
    for (int u0 = 0; u0 < n; u0 += VPW)
    {
        const int u = u0 + sub;
        bool live = u < n;
        const int j = u < ns ? u : lo + u - ns;
        float k[E] = {}, v[E] = {}, ks = 1.f, vs = 1.f;
        if (live)
        {
            const int pg = __ldg(a.b.table + s * a.b.table_stride + j / a.c.page_size);
            const int in = j % a.c.page_size;
            if (pg < 0 || pg >= a.c.num_pages)
            {
                paged_status(a.c.status, kPagedBadPage);
                live = false;
            }
            else
            {
                const long long at = pg * a.c.page_stride + in * a.c.row_stride + g * a.c.head_stride + d;
                load_row<CT, E>(a.c.k, at, k);
                load_row<CT, E>(a.c.v, at, v);
                if constexpr (kCodes<CT>)
                {
                    const long long sa = pg * a.c.s_page_stride + in * a.c.s_row_stride + g * a.c.s_head_stride;
                    ks = __ldg(a.c.k_scale + sa);
                    vs = __ldg(a.c.v_scale + sa);
                }
            }
        }
        float sc = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) sc += q[i] * k[i];
#pragma unroll
        for (int o = LPV / 2; o > 0; o >>= 1) sc += __shfl_xor_sync(0xffffffffu, sc, o);
        if (!live) continue;
        sc *= ks * a.scale_log2;
        const float mn = fmaxf(m, sc);
        const float corr = m == mn ? 1.f : exp2f(m - mn), e = sc == -INFINITY ? 0.f : exp2f(sc - mn);   // a NaN stays one
        l = l * corr + e;
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] = acc[i] * corr + e * vs * v[i];
        m = mn;
    }
    // The VPW parts of a warp (each saw every VPW-th key) into one.
    float M = m;
#pragma unroll
    for (int o = LPV; o < 32; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float f = m == M ? 1.f : exp2f(m - M);
    l *= f;
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] *= f;
#pragma unroll
    for (int o = LPV; o < 32; o <<= 1)
    {
        l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
    }
    if (sub) return;
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = l == 0.f ? 0.f : acc[i] / l;
    store_row<QT, E>(a.out, r * a.o_row_stride + h * a.o_head_stride + d, acc);
}

}  // namespace hy
