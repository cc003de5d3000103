// Norms of query and key heads with the position rotation in the same pass, from
// row tensors to row tensors or, for k and v, into the paged cache.
//
// A head is D numbers x; with the row's c and s it becomes w y / sqrt(mean(y^2) + eps),
// y = turn(x) (rotation first), or turn(w x) / sqrt(mean(x^2) + eps) (norm first: the
// rotation is linear, so the row's one factor can be taken out of it). Both
// halves of a head meet in the rotation, so a lane holds a 16-byte piece of the
// first half and the piece that belongs to it of the second: the rotation stays in
// the lane, and the mean is a sum over the head's 4, 8 or 16 lanes.
//
// Memory bounds it: every row is read once and written once. A warp takes a
// row's heads one group after another, so that the row's angles (which are as
// many bytes as two heads of fp32) are loaded once and stay in registers; a row
// is split over the warps of a CTA, and over several CTAs, only while there are too
// few rows to fill the GPU.
#pragma once

#include "hy_paged.cuh"

namespace hy {

struct RotateArgs {
    const void* q;
    const void* k;
    const void* v;   // cache form
    void* q_out;
    void* k_out;     // row form
    long long q_row, q_head, k_row, k_head, v_row, v_head, qo_row, qo_head, ko_row, ko_head;
    const float* q_weight;
    const float* k_weight;
    const float* cos;
    const float* sin;
    const int* positions;
    long long table_stride;
    int table_rows;
    float eps, inv_dim;
    int rotate_first;
    int rows, q_heads, kv_heads;
    int per_cta;          // rows of a CTA, at most kRowsPerCta
    int whole;            // a warp takes a whole row; else the CTA's (and gridDim.y CTAs') warps share each
    int* status;
    PagedCache c;         // cache form
    PagedBatch b;
};

template <typename RT, typename CT, int D, bool CACHE>
__global__ void __launch_bounds__(kRowWarps * 32) rotate_kernel(const RotateArgs a)
{
    constexpr int E = 16 / static_cast<int>(sizeof(RT));   // elements of a piece
    constexpr int LPV = D / (2 * E);                       // lanes per head: 4, 8 or 16
    constexpr int VPW = 32 / LPV;                          // heads per warp and step
    constexpr int U = 2;                                   // steps in flight
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / LPV, d = (lane % LPV) * E;
    const int r0 = blockIdx.x * a.per_cta, n_rows = min(a.per_cta, a.rows - r0);
    const int nv = a.q_heads + (CACHE ? 2 : 1) * a.kv_heads;
    const int stride = a.whole ? VPW : kRowWarps * static_cast<int>(gridDim.y) * VPW;
    const int v_first = a.whole ? 0 : (static_cast<int>(blockIdx.y) * kRowWarps + warp) * VPW;
    __shared__ PagedPlace places[kRowsPerCta];
    pdl_wait();
    if constexpr (CACHE) paged_places(a.c, a.b, r0, n_rows, places);

    for (int i = a.whole ? warp : 0; i < n_rows; i += a.whole ? kRowWarps : 1)
    {
        const int r = r0 + i;
        PagedPlace place = {0, 0};
        if constexpr (CACHE)
        {
            place = places[i];
            if (place.off == -1) continue;   // (uniform in the warp)
        }
        // Heads x: q, then k, then (cache form) v.
        auto at = [&](int x) -> const RT* {
            const RT* p;
            if (x < a.q_heads) p = static_cast<const RT*>(a.q) + r * a.q_row + x * a.q_head;
            else if (!CACHE || x < a.q_heads + a.kv_heads) p = static_cast<const RT*>(a.k) + r * a.k_row + (x - a.q_heads) * a.k_head;
            else p = static_cast<const RT*>(a.v) + r * a.v_row + (x - a.q_heads - a.kv_heads) * a.v_head;
            return p + d;
        };
        uint4 next[U][2];
        auto load = [&](int x0) {
#pragma unroll
            for (int u = 0; u < U; ++u)
            {
                const int x = x0 + u * stride + sub;
                if (x >= nv) continue;
                const RT* const p = at(x);
                next[u][0] = *reinterpret_cast<const uint4*>(p);   // (not __ldg: the outputs may lie in the same place)
                next[u][1] = *reinterpret_cast<const uint4*>(p + D / 2);
            }
        };
        load(v_first);
        float cs[2][E], sn[2][E];   // the row's angles, both pieces
        {
            const int t = a.positions ? __ldg(a.positions + r) : r;
            if (t >= 0 && t < a.table_rows)
            {
#pragma unroll
                for (int p = 0; p < 2; ++p)
                {
                    load_row<float, E>(a.cos, t * a.table_stride + d + p * (D / 2), cs[p]);
                    load_row<float, E>(a.sin, t * a.table_stride + d + p * (D / 2), sn[p]);
                }
            }
            else
            {
                if (lane == 0) paged_status(a.status, kPagedBadPosition);
#pragma unroll
                for (int e = 0; e < E; ++e) cs[0][e] = cs[1][e] = sn[0][e] = sn[1][e] = __int_as_float(0x7fffffff);
            }
        }
        float w[2][E];        // weights of the kind of head that came last
        int kind_w = -1;
        for (int x0 = v_first; x0 < nv; x0 += U * stride)
        {
            uint4 raw[U][2];
#pragma unroll
            for (int u = 0; u < U; ++u)
            {
                raw[u][0] = next[u][0];
                raw[u][1] = next[u][1];
            }
            if (x0 + U * stride < nv) load(x0 + U * stride);
#pragma unroll
            for (int u = 0; u < U; ++u)
            {
                const int x = x0 + u * stride + sub;
                const bool live = x < nv;
                const int kind = x < a.q_heads ? 0 : (!CACHE || x < a.q_heads + a.kv_heads) ? 1 : 2;
                float f[2][E];
#pragma unroll
                for (int p = 0; p < 2; ++p)
                {
                    const uint32_t w4[4] = {raw[u][p].x, raw[u][p].y, raw[u][p].z, raw[u][p].w};
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        f[p][e] = E == 4 ? __uint_as_float(w4[e]) : __uint_as_float((e & 1) ? w4[e >> 1] & 0xFFFF0000u : w4[e >> 1] << 16);
                }
                if (kind < 2 && live && kind != kind_w)
                {
#pragma unroll
                    for (int p = 0; p < 2; ++p) load_row<float, E>(kind ? a.k_weight : a.q_weight, d + p * (D / 2), w[p]);
                    kind_w = kind;
                }
                if (kind < 2)
                {
                    float ss = 0.f;
                    auto squares = [&] {
#pragma unroll
                        for (int e = 0; e < E; ++e) ss = fmaf(f[0][e], f[0][e], fmaf(f[1][e], f[1][e], ss));
                    };
                    auto weigh = [&] {
#pragma unroll
                        for (int e = 0; e < E; ++e)
                        {
                            f[0][e] *= w[0][e];
                            f[1][e] *= w[1][e];
                        }
                    };
                    if (!a.rotate_first)
                    {
                        squares();
                        weigh();
                    }
#pragma unroll
                    for (int e = 0; e < E; ++e)
                    {
                        const float lo = f[0][e], hi = f[1][e];
                        f[0][e] = fmaf(lo, cs[0][e], -hi * sn[0][e]);
                        f[1][e] = fmaf(hi, cs[1][e], lo * sn[1][e]);
                    }
                    if (a.rotate_first)
                    {
                        squares();
                        weigh();
                    }
                    // (lanes of one head agree on `kind`, and the shuffles stay within them)
                    const unsigned mates = (LPV == 32 ? 0xffffffffu : ((1u << LPV) - 1u)) << (sub * LPV);
#pragma unroll
                    for (int o = LPV / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mates, ss, o);
                    const float factor = rsqrtf(fmaf(ss, a.inv_dim, a.eps));
#pragma unroll
                    for (int e = 0; e < E; ++e)
                    {
                        f[0][e] *= factor;
                        f[1][e] *= factor;
                    }
                }
                if (!CACHE || kind == 0)
                {
                    if (!live) continue;
                    const int h = kind ? x - a.q_heads : x;
                    RT* const o = static_cast<RT*>(kind ? a.k_out : a.q_out) + (kind ? r * a.ko_row + h * a.ko_head : r * a.qo_row + h * a.qo_head) + d;
                    store_row<RT, E>(o, 0, f[0]);
                    store_row<RT, E>(o, D / 2, f[1]);
                }
                else if constexpr (CACHE)
                {
                    const int h = x - a.q_heads - (kind == 2 ? a.kv_heads : 0);
                    const bool put = live && place.off >= 0;
                    const long long to = place.off + h * a.c.head_stride + d;
                    void* const pool = kind == 2 ? a.c.v : a.c.k;
                    if constexpr (kCodes<CT>)
                    {
                        // The largest magnitude by its bits: an infinity or a NaN comes out on top.
                        uint32_t m = 0;
#pragma unroll
                        for (int e = 0; e < E; ++e) m = max(m, max(__float_as_uint(f[0][e]) & 0x7fffffffu, __float_as_uint(f[1][e]) & 0x7fffffffu));
                        const unsigned mates = ((1u << LPV) - 1u) << (sub * LPV);
#pragma unroll
                        for (int o = LPV / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(mates, m, o));
                        if (!put) continue;
                        const bool finite = m < 0x7f800000u;
                        const float scale = finite ? code_scale<CT>(__uint_as_float(m)) : __int_as_float(0x7fffffff);
                        const float inv = __fdividef(1.f, scale);   // (scale < 2^126; off by 2 ulp, which quant4 allows for)
                        uint8_t* const o = static_cast<uint8_t*>(pool) + to;
#pragma unroll
                        for (int p = 0; p < 2; ++p)
                        {
                            uint32_t c4[E / 4];
#pragma unroll
                            for (int y = 0; y < E / 4; ++y) c4[y] = finite ? quant4<CT>(f[p] + 4 * y, scale, inv) : 0u;
                            if constexpr (E == 8) *reinterpret_cast<uint2*>(o + p * (D / 2)) = make_uint2(c4[0], c4[1]);
                            else *reinterpret_cast<uint32_t*>(o + p * (D / 2)) = c4[0];
                        }
                        if (lane % LPV == 0) (kind == 2 ? a.c.v_scale : a.c.k_scale)[place.s_off + h * a.c.s_head_stride] = scale;
                    }
                    else if (put)
                    {
                        store_row<CT, E>(pool, to, f[0]);
                        store_row<CT, E>(pool, to + D / 2, f[1]);
                    }
                }
            }
        }
    }
}

}  // namespace hy
