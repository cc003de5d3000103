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
// many bytes as two heads of fp32) are loaded once and stay in registers; they and
// the heads come through a ring of the warp's own in shared memory, four steps of 1 KB
// ahead and across rows (with loads into registers, one step ahead, too little was in flight). A row
// is split over the warps of a CTA, and over several CTAs, only while there are too
// few rows to fill the GPU. 20011 bf16 rows of 36 heads of 64: 38 us, 5.0 TB/s (62 us with loads into registers);
// 38.6k bf16 rows of 32 heads of 128, k and v into E4M3 pages: 131 us, 4.4 TB/s. What bounds that one is a warp's chain of
// shared-memory loads, two reductions over a head's lanes, divide, quantise and store, with too few warps to hide it: four
// CTAs of four per SM (122 registers; shared memory allows no more either), 59% of the issue slots, and of a warp's time
// hardly any waits for memory. With five CTAs the registers spill: 150 us. One fp32 row: 1.7 us.
#pragma once

#include "hy_paged_attn.cuh"

namespace hy {

constexpr int kRotateRing = 4;   // steps of a warp's ring

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
    int rows, q_heads, kv_heads;
    int per_cta;          // rows of a CTA, at most kRowsPerCta
    int whole;            // a warp takes a whole row; else the CTA's (and gridDim.y CTAs') warps share each
    int* status;
    PagedCache c;         // cache form
    PagedBatch b;
};

// E floats as pairs.
template <int E>
__device__ __forceinline__ void load_pairs(const float* p, uint64_t (&o)[E / 2])
{
#pragma unroll
    for (int e = 0; e < E; e += 4)
    {
        const float4 x = __ldg(reinterpret_cast<const float4*>(p + e));
        o[e / 2] = f2(x.x, x.y);
        o[e / 2 + 1] = f2(x.z, x.w);
    }
}

template <typename RT, typename CT, int D, bool CACHE, bool FIRST>   // FIRST: rotation first
__global__ void __launch_bounds__(kRowWarps * 32, CACHE ? 4 : 5) rotate_kernel(const RotateArgs a)
{
    constexpr int E = 16 / static_cast<int>(sizeof(RT));   // elements of a piece
    constexpr int H = E / 2;                               // pairs
    constexpr int LPV = D / (2 * E);                       // lanes per head: 4, 8 or 16
    constexpr int VPW = 32 / LPV;                          // heads per warp and step
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / LPV, d = (lane % LPV) * E;
    const unsigned mates = ((1u << LPV) - 1u) << (sub * LPV);   // lanes of a head: they agree in all that is decided
    const int r0 = blockIdx.x * a.per_cta, n_rows = min(a.per_cta, a.rows - r0);
    const int nv = a.q_heads + (CACHE ? 2 : 1) * a.kv_heads;
    const int stride = a.whole ? VPW : kRowWarps * static_cast<int>(gridDim.y) * VPW;
    const int v_first = a.whole ? 0 : (static_cast<int>(blockIdx.y) * kRowWarps + warp) * VPW;
    const int steps = max(0, (nv - v_first + stride - 1) / stride);             // of a row
    const int row_first = a.whole ? warp : 0, row_step = a.whole ? kRowWarps : 1;
    const int total = max(0, (n_rows - row_first + row_step - 1) / row_step) * steps;
    __shared__ PagedPlace places[kRowsPerCta];
    __shared__ __align__(16) uint4 ring[kRowWarps][kRotateRing][2][32];          // [step][piece][lane]
    __shared__ __align__(16) float angles[kRowWarps][kRotateRing][2][D];         // [row][cos, sin]
    pdl_wait();
    // Table rows of the CTA's rows, a lane's each.
    const int table_row = lane >= n_rows ? -1 : a.positions ? __ldg(a.positions + r0 + lane) : r0 + lane;
    int fi = 0, fx = 0, ft = 0;   // row, step of it and step in all that is fetched next
    auto fetch = [&] {
        if (ft < total)
        {
            const int i = row_first + fi * row_step, r = r0 + i, x = v_first + fx * stride + sub;
            if (x < nv)
            {
                // Heads x: q, then k, then (cache form) v.
                const RT* const p = (x < a.q_heads                          ? static_cast<const RT*>(a.q) + r * a.q_row + x * a.q_head
                                     : !CACHE || x < a.q_heads + a.kv_heads ? static_cast<const RT*>(a.k) + r * a.k_row + (x - a.q_heads) * a.k_head
                                                                            : static_cast<const RT*>(a.v) + r * a.v_row + (x - a.q_heads - a.kv_heads) * a.v_head) + d;
                const uint32_t to = smem_u32(&ring[warp][ft % kRotateRing][0][lane]);
                cp_async16_zfill(to, p, true);
                cp_async16_zfill(to + 512, p + D / 2, true);
            }
            if (fx == 0)
            {
                const int t = __shfl_sync(0xffffffffu, table_row, i);
                if (t >= 0 && t < a.table_rows)
#pragma unroll
                    for (int y = lane; y < D / 2; y += 32)   // 16-byte pieces of both
                        cp_async16_zfill(smem_u32(&angles[warp][fi % kRotateRing][0][0]) + y * 16,
                                         (y < D / 4 ? a.cos : a.sin) + t * a.table_stride + y % (D / 4) * 4, true);
            }
            if (++fx == steps)
            {
                fx = 0;
                ++fi;
            }
            ++ft;
        }
        cp_commit();
    };
#pragma unroll
    for (int y = 0; y < kRotateRing - 1; ++y) fetch();
    if constexpr (CACHE) paged_places(a.c, a.b, r0, n_rows, places);

    uint64_t w[2][H];     // weights of the kind of head that came last
    int kind_w = -1, done = 0;
    for (int i = row_first, row_no = 0; done < total; i += row_step, ++row_no)
    {
        const int r = r0 + i;
        PagedPlace place = {0, 0};
        if constexpr (CACHE) place = places[i];
        uint64_t cs[2][H], sn[2][H];   // the row's angles, both pieces; the first sine negated
        for (int step = 0; step < steps; ++step, ++done)
        {
            cp_wait<kRotateRing - 2>();
            __syncwarp();
            fetch();
            const int x = v_first + step * stride + sub;
            if (step == 0)
            {
                const int t = __shfl_sync(0xffffffffu, table_row, i);
                if (t >= 0 && t < a.table_rows)
                {
                    const float* const at = &angles[warp][row_no % kRotateRing][0][d];
#pragma unroll
                    for (int p = 0; p < 2; ++p)
#pragma unroll
                        for (int e = 0; e < E; e += 4)
                        {
                            const float4 c = *reinterpret_cast<const float4*>(at + p * (D / 2) + e), n = *reinterpret_cast<const float4*>(at + D + p * (D / 2) + e);
                            cs[p][e / 2] = f2(c.x, c.y);
                            cs[p][e / 2 + 1] = f2(c.z, c.w);
                            sn[p][e / 2] = f2(n.x, n.y);
                            sn[p][e / 2 + 1] = f2(n.z, n.w);
                        }
#pragma unroll
                    for (int e = 0; e < H; ++e) sn[0][e] ^= 0x8000000080000000ull;
                }
                else
                {
                    if (lane == 0 && place.off != -1) paged_status(a.status, kPagedBadPosition);
#pragma unroll
                    for (int e = 0; e < H; ++e) cs[0][e] = cs[1][e] = sn[0][e] = sn[1][e] = 0x7fffffff7fffffffull;   // NaN
                }
            }
            if (x >= nv || (CACHE && place.off == -1)) continue;   // (alike for a head's lanes)
            const uint4 y0 = ring[warp][done % kRotateRing][0][lane], y1 = ring[warp][done % kRotateRing][1][lane];
            const uint32_t raw[2][4] = {{y0.x, y0.y, y0.z, y0.w}, {y1.x, y1.y, y1.z, y1.w}};
            const int kind = x < a.q_heads ? 0 : (!CACHE || x < a.q_heads + a.kv_heads) ? 1 : 2;
            uint64_t f[2][H];
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int e = 0; e < H; ++e)
                    f[p][e] = E == 4 ? f2(__uint_as_float(raw[p][2 * e]), __uint_as_float(raw[p][2 * e + 1]))
                                     : f2(__uint_as_float(raw[p][e] << 16), __uint_as_float(raw[p][e] & 0xFFFF0000u));
            if (kind < 2)
            {
                if (kind != kind_w)
                {
#pragma unroll
                    for (int p = 0; p < 2; ++p) load_pairs<E>((kind ? a.k_weight : a.q_weight) + d + p * (D / 2), w[p]);
                    kind_w = kind;
                }
                uint64_t ss = 0;   // (a pair of zeros)
                auto squares = [&] {
#pragma unroll
                    for (int e = 0; e < H; ++e) ss = f2_fma(f[0][e], f[0][e], f2_fma(f[1][e], f[1][e], ss));
                };
                auto weigh = [&] {
#pragma unroll
                    for (int e = 0; e < H; ++e)
                    {
                        f[0][e] = f2_mul(f[0][e], w[0][e]);
                        f[1][e] = f2_mul(f[1][e], w[1][e]);
                    }
                };
                if constexpr (!FIRST)
                {
                    squares();
                    weigh();
                }
#pragma unroll
                for (int e = 0; e < H; ++e)
                {
                    const uint64_t lo = f[0][e], hi = f[1][e];
                    f[0][e] = f2_fma(lo, cs[0][e], f2_mul(hi, sn[0][e]));
                    f[1][e] = f2_fma(hi, cs[1][e], f2_mul(lo, sn[1][e]));
                }
                if constexpr (FIRST)
                {
                    squares();
                    weigh();
                }
                float s0, s1;
                f2_get(ss, s0, s1);
                s0 += s1;
#pragma unroll
                for (int o = LPV / 2; o > 0; o >>= 1) s0 += __shfl_xor_sync(mates, s0, o);
                const float factor = rsqrtf(fmaf(s0, a.inv_dim, a.eps));
                const uint64_t factor2 = f2(factor, factor);
#pragma unroll
                for (int e = 0; e < H; ++e)
                {
                    f[0][e] = f2_mul(f[0][e], factor2);
                    f[1][e] = f2_mul(f[1][e], factor2);
                }
            }
            float o[2][E];
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int e = 0; e < H; ++e) f2_get(f[p][e], o[p][2 * e], o[p][2 * e + 1]);
            if (!CACHE || kind == 0)
            {
                const int h = kind ? x - a.q_heads : x;
                RT* const to = static_cast<RT*>(kind ? a.k_out : a.q_out) + (kind ? r * a.ko_row + h * a.ko_head : r * a.qo_row + h * a.qo_head) + d;
                store_row<RT, E>(to, 0, o[0]);
                store_row<RT, E>(to, D / 2, o[1]);
            }
            else if constexpr (CACHE)
            {
                if (place.off < 0) continue;   // (uniform in the warp)
                const int h = x - a.q_heads - (kind == 2 ? a.kv_heads : 0);
                const long long to = place.off + h * a.c.head_stride + d;
                void* const pool = kind == 2 ? a.c.v : a.c.k;
                if constexpr (kCodes<CT>)
                {
                    // The largest magnitude by its bits: an infinity or a NaN comes out on top.
                    uint32_t m = 0;
#pragma unroll
                    for (int e = 0; e < E; ++e) m = max(m, max(__float_as_uint(o[0][e]) & 0x7fffffffu, __float_as_uint(o[1][e]) & 0x7fffffffu));
#pragma unroll
                    for (int y = LPV / 2; y > 0; y >>= 1) m = max(m, __shfl_xor_sync(mates, m, y));
                    const bool finite = m < 0x7f800000u;
                    const float scale = finite ? code_scale<CT>(__uint_as_float(m)) : __int_as_float(0x7fffffff);
                    const float inv = __fdividef(1.f, scale);   // (scale < 2^126; off by 2 ulp, which quant4 allows for)
                    uint8_t* const b = static_cast<uint8_t*>(pool) + to;
#pragma unroll
                    for (int p = 0; p < 2; ++p)
                    {
                        uint32_t c4[E / 4];
#pragma unroll
                        for (int y = 0; y < E / 4; ++y) c4[y] = finite ? quant4<CT>(o[p] + 4 * y, scale, inv) : 0u;
                        if constexpr (E == 8) *reinterpret_cast<uint2*>(b + p * (D / 2)) = make_uint2(c4[0], c4[1]);
                        else *reinterpret_cast<uint32_t*>(b + p * (D / 2)) = c4[0];
                    }
                    if (lane % LPV == 0) (kind == 2 ? a.c.v_scale : a.c.k_scale)[place.s_off + h * a.c.s_head_stride] = scale;
                }
                else
                {
                    store_row<CT, E>(pool, to, o[0]);
                    store_row<CT, E>(pool, to + D / 2, o[1]);
                }
            }
        }
    }
}

}  // namespace hy
