// Paged KV cache: rows written into pages (quantised as they are written) and
// read back. The attention over the pages is in hy_paged_attn.cuh.
//
// A batch names its sequences by device arrays: the row range q_start[s] ..
// q_start[s + 1], the cache length kv_len[s] (the new rows included) and a row
// of page numbers; every kernel checks what it reads from them and skips what
// does not hold, setting a bit of the status word.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "hy_device.cuh"

namespace hy {

// Status bits (enum hy_paged_status).
constexpr int kPagedBadPage = 1;
constexpr int kPagedBadLength = 2;
constexpr int kPagedBadRows = 4;
constexpr int kPagedTimeout = 8;
constexpr int kPagedBadPosition = 16;

struct PagedCache {
    void* k;
    void* v;
    float* k_scale;   // 8-bit caches
    float* v_scale;
    long long page_stride, head_stride, row_stride;      // elements
    long long s_page_stride, s_head_stride, s_row_stride;
    int num_pages, page_size, kv_heads;
    int* status;
};

struct PagedBatch {
    const int* q_start;
    const int* kv_len;
    const int* table;
    long long table_stride;
    int table_width, num_seqs, rows;
};

__device__ __forceinline__ void paged_status(int* status, int bit)
{
    if (status) atomicOr(status, bit);
}

// Rows and cache length of sequence s; false (and a status bit) when they do not hold.
struct PagedSeq {
    int row0, n, kv;
};
__device__ __forceinline__ bool paged_seq(const PagedBatch& b, int s, int page_size, int* status, PagedSeq& o)
{
    const int r0 = __ldg(b.q_start + s), r1 = __ldg(b.q_start + s + 1), kv = __ldg(b.kv_len + s);
    o.row0 = r0;
    o.n = r1 - r0;
    o.kv = kv;
    if (r0 < 0 || r1 < r0 || r1 > b.rows)
    {
        paged_status(status, kPagedBadRows);
        return false;
    }
    if (kv < 0 || kv > static_cast<long long>(b.table_width) * page_size)
    {
        paged_status(status, kPagedBadLength);
        return false;
    }
    return true;
}

// The sequence that holds row r (the last one whose q_start is <= r), by the
// whole warp: 32 starts per round, counted by a ballot. -1: r lies before the first sequence;
// num_seqs: behind the last.
__device__ __forceinline__ int paged_find_seq(const PagedBatch& b, int r, int lane)
{
    int below = 0;
    for (int s0 = 0; s0 <= b.num_seqs; s0 += 32)
    {
        const int s = s0 + lane;
        const bool le = s <= b.num_seqs && __ldg(b.q_start + s) <= r;
        const int c = __popc(__ballot_sync(0xffffffffu, le));
        below += c;
        if (c < 32) break;
    }
    return below - 1;
}

// ---------------------------------------------------------------------------
// Element types of the cache.
// ---------------------------------------------------------------------------
struct E4M3 {
    uint8_t c;
};
struct Int8 {
    uint8_t c;
};
template <typename CT>
constexpr bool kCodes = (sizeof(CT) == 1);   // codes with a scale

// x / s rounded to fp32 so that no later rounding to fewer bits can go wrong: where the quotient is not a
// float, of the two floats around it the one whose last bit is set (it lies on the quotient's side
// of every tie). The remainder x - q s of the nearest q is exact in a fused multiply-add as long as it is no
// smaller than the smallest number: scales below 2^-60 and their x are first taken 2^80 times (exactly; a
// quotient next to a tie is at least 2^-10, so its remainder is a multiple of 2^(-33 - 23 - 60)).
__device__ __forceinline__ float quotient_odd(float x, float s, float inv)
{
    const bool tiny = s < 0x1p-60f;
    x *= tiny ? 0x1p80f : 1.f;
    s *= tiny ? 0x1p80f : 1.f;
    inv *= tiny ? 0x1p-80f : 1.f;
    float q = x * inv;
    q = fmaf(fmaf(-q, s, x), inv, q);
    const float r = fmaf(-q, s, x);
    const int bits = __float_as_int(q);
    const int away = ((__float_as_int(r) ^ bits) < 0) ? -1 : 1;   // the quotient is the smaller or the larger magnitude
    return __int_as_float((r == 0.f || (bits & 1) || (bits << 1) == 0) ? bits : bits + away);
}

// Two fp32 at once.
__device__ __forceinline__ uint64_t f2(float x, float y)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void f2_get(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Four quotients x / s as a word of codes, rounded to nearest, ties to even (inv = 1 / s, off by 2 ulp at
// most): the hardware's rounding of a product that is surely a little below the quotient and of one that is a
// little above (lo and hi: inv (1 -+ 2^-20)). Rounding is monotone, so equal codes are the quotient's; else a tie may lie between, and
// quotient_odd decides. (bf16 rows meet ties often: one in some 300 quotients of 8-bit significands is within
// rounding of one. Looking for ties in the quotient's bits took three times the integer instructions, which bound it.)
template <typename CT>
__device__ __forceinline__ uint32_t quant4(const float* x, float s, float inv)
{
    const float lo = inv * (1.f - 0x1p-20f), hi = inv * (1.f + 0x1p-20f);
    auto codes = [](const float* q) {
        uint32_t w;
        if constexpr (std::is_same_v<CT, E4M3>)
            asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
                "mov.b32 %0, {lo, hi};\n\t}"
                : "=r"(w)
                : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]));
        else   // (q holds integers plus 1.5 * 2^23)
            w = __byte_perm(__byte_perm(__float_as_uint(q[0]), __float_as_uint(q[1]), 0x0040),
                            __byte_perm(__float_as_uint(q[2]), __float_as_uint(q[3]), 0x0040), 0x5410);
        return w;
    };
    // x times f; INT8: to an integer by adding 1.5 * 2^23 in the same rounding; magnitudes stay within 127 (1 + 2^-19).
    auto times = [&](float f, float* q) {
#pragma unroll
        for (int e = 0; e < 4; e += 2)
            f2_get(std::is_same_v<CT, E4M3> ? f2_mul(f2(x[e], x[e + 1]), f2(f, f))
                                            : f2_fma(f2(x[e], x[e + 1]), f2(f, f), f2(12582912.f, 12582912.f)),
                   q[e], q[e + 1]);
    };
    float q[4], p[4];
    times(lo, q);
    times(hi, p);
    uint32_t w = codes(q);
    if (w != codes(p))
    {
#pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            q[e] = quotient_odd(x[e], s, inv);
            if constexpr (!std::is_same_v<CT, E4M3>) q[e] += 12582912.f;
        }
        w = codes(q);
    }
    return w;
}
template <typename CT>
constexpr float kCodeMax = std::is_same_v<CT, E4M3> ? 448.f : 127.f;

// m / kCodeMax correctly rounded, at least 2^-126: the quotient by the rounded reciprocal and its
// exact remainder once more (Markstein); below 2^-126 kCodeMax, where that could underflow, the bound applies.
template <typename CT>
__device__ __forceinline__ float code_scale(float m)
{
    constexpr float top = kCodeMax<CT>, inv = 1.f / top;
    const float q = m * inv;
    return fmaxf(fmaf(fmaf(-q, top, m), inv, q), 1.17549435e-38f);
}

// Four codes of a word as fp32.
template <typename CT>
__device__ __forceinline__ void decode4(uint32_t w, float* o)
{
    if constexpr (std::is_same_v<CT, E4M3>)
    {
        uint32_t h0, h1;
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
            : "=r"(h0), "=r"(h1)
            : "r"(w));
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h0)), b = __half22float2(*reinterpret_cast<const __half2*>(&h1));
        o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y;
    }
    else
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
    }
}

// E consecutive elements (E = 4 or 8) at p as fp32, by the widest loads; stores likewise.
template <typename T, int E>
__device__ __forceinline__ void load_row(const void* base, long long off, float* x)
{
    if constexpr (sizeof(T) == 4)
    {
#pragma unroll
        for (int i = 0; i < E; i += 4)
        {
            const float4 f = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(base) + off + i));
            x[i] = f.x; x[i + 1] = f.y; x[i + 2] = f.z; x[i + 3] = f.w;
        }
    }
    else if constexpr (sizeof(T) == 2)
    {
        uint32_t w[E / 2];
        const uint16_t* p = static_cast<const uint16_t*>(base) + off;
        if constexpr (E == 8)
        {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
            w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
        }
        else
        {
            const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
            w[0] = u.x; w[1] = u.y;
        }
#pragma unroll
        for (int i = 0; i < E / 2; ++i)
        {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    else
    {
        const uint8_t* p = static_cast<const uint8_t*>(base) + off;
        if constexpr (E == 8)
        {
            const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
            decode4<T>(u.x, x);
            decode4<T>(u.y, x + 4);
        }
        else
        {
            decode4<T>(__ldg(reinterpret_cast<const uint32_t*>(p)), x);
        }
    }
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T, int E>   // fp32 or bf16
__device__ __forceinline__ void store_row(void* base, long long off, const float* x)
{
    if constexpr (sizeof(T) == 4)
    {
#pragma unroll
        for (int i = 0; i < E; i += 4)
            *reinterpret_cast<float4*>(static_cast<float*>(base) + off + i) =
                make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    }
    else
    {
        uint16_t* p = static_cast<uint16_t*>(base) + off;
        if constexpr (E == 8)
            *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]),
                                                      pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
        else
            *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
    }
}

// ---------------------------------------------------------------------------
// Write and read back. A CTA of 4 warps takes a few consecutive rows (1 to 16, so
// that small calls spread over the SMs and in large ones a place is looked up
// once for all that is moved): lane r of every warp finds row r's page, then the
// rows' 2 x kv_heads vectors (k, then v) are shared out to groups of lanes that
// hold two pieces of 16 bytes of the row tensor each, so that all loads are wide, several
// are in flight per lane and the index arithmetic serves 32 bytes (with one piece both calls
// on the 38.6k rows below took 113 us, with two 99). The maximum of a vector is taken in registers and its codes
// leave in the same pass. Each byte moves once: reading 264k rows of 8 heads of 128 (INT8
// to bf16) takes 290 us, 6.0 TB/s; writing 38.6k such rows (bf16 to E4M3) 62 us, reading them
// back 42 us; the write is bound by its instructions (69% of the issue slots, integer units 63%
// busy) rather than by its 237 MB.
// ---------------------------------------------------------------------------
constexpr int kRowWarps = 4;
constexpr int kRowsPerCta = 16;

struct PagedRowArgs {
    PagedCache c;
    PagedBatch b;
    void* k;   // row tensors
    void* v;
    int k_row_stride, k_head_stride, v_row_stride, v_head_stride;
    int page_head_stride, scale_head_stride;   // the cache's
    int per_cta;               // rows of a CTA
    unsigned vectors_inv;      // ceil(2^32 / (2 kv_heads)): x / (2 kv_heads) = high half of the product, x < 2^16
};

// Where a CTA's rows belong: offsets of the page and the row in it, for the elements and for the scales.
constexpr long long kPlaceLost = -2;
struct PagedPlace {
    long long off, s_off;   // off < 0: nowhere (kPlaceLost: a row of a sequence, but its page is not one)
};
// The place of row r (r < 0: none), by a whole warp, a consecutive row for each of its lanes.
__device__ __forceinline__ void paged_find_place(const PagedCache& c, const PagedBatch& b, int r, int lane, PagedPlace& o)
{
    o.off = -1;
    o.s_off = 0;
    int s = paged_find_seq(b, __shfl_sync(0xffffffffu, r, 0), lane);   // of the first row
    if (r < 0 || r >= b.rows) return;
    s = max(s, 0);
    while (s < b.num_seqs && __ldg(b.q_start + s + 1) <= r) ++s;       // (rows of short sequences)
    if (s >= b.num_seqs || r < __ldg(b.q_start + s)) return;
    PagedSeq q;
    if (!paged_seq(b, s, c.page_size, c.status, q)) return;
    if (r < q.row0 || r >= q.row0 + q.n)   // q_start is not ascending
    {
        paged_status(c.status, kPagedBadRows);
        return;
    }
    const int p = q.kv - q.n + (r - q.row0);
    if (p < 0) return;
    const int x = p / c.page_size, in = p - x * c.page_size;
    const int pg = __ldg(b.table + s * b.table_stride + x);
    if (pg < 0 || pg >= c.num_pages)
    {
        paged_status(c.status, kPagedBadPage);
        o.off = kPlaceLost;
        return;
    }
    o.off = pg * c.page_stride + in * c.row_stride;
    o.s_off = pg * c.s_page_stride + in * c.s_row_stride;
}
__device__ __forceinline__ void paged_places(const PagedCache& c, const PagedBatch& b, int r0, int n_rows, PagedPlace* places)
{
    if (threadIdx.x < 32)
    {
        const int lane = threadIdx.x;
        PagedPlace o;
        paged_find_place(c, b, lane < n_rows ? r0 + lane : -1, lane, o);
        if (lane < kRowsPerCta) places[lane] = o;
    }
    __syncthreads();
}

// Vector x of a CTA's rows: row x / (2 kv_heads), k or v, head.
struct PagedVector {
    int row, head;
    bool isv;
};
__device__ __forceinline__ PagedVector paged_vector(const PagedRowArgs& a, int x)
{
    const int row = static_cast<int>(__umulhi(static_cast<unsigned>(x), a.vectors_inv));
    const int y = x - row * 2 * a.c.kv_heads;
    const bool isv = y >= a.c.kv_heads;
    return {row, isv ? y - a.c.kv_heads : y, isv};
}
template <typename RT>
__device__ __forceinline__ RT* paged_row_at(const PagedRowArgs& a, const PagedVector& v, int r0)
{
    RT* const p = static_cast<RT*>(v.isv ? a.v : a.k) + static_cast<long long>(r0 + v.row) * (v.isv ? a.v_row_stride : a.k_row_stride);
    return p + static_cast<long long>(v.head) * (v.isv ? a.v_head_stride : a.k_head_stride);
}

template <typename RT, typename CT, int D>
__global__ void __launch_bounds__(kRowWarps * 32) paged_write_kernel(const PagedRowArgs a)
{
    constexpr int E = 16 / static_cast<int>(sizeof(RT));   // elements of a piece
    constexpr int P = 2;                                   // pieces per lane, D / P elements apart
    constexpr int LPV = D / (E * P);                       // lanes per vector: 4, 8 or 16
    constexpr int VPW = 32 / LPV;                          // vectors per warp and step
    constexpr int U = 2;                                   // steps in flight
    constexpr int STEP = U * kRowWarps * VPW;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r0 = blockIdx.x * a.per_cta, n_rows = min(a.per_cta, a.b.rows - r0);
    const int nv = n_rows * 2 * a.c.kv_heads, sub = lane / LPV, d = (lane % LPV) * E;
    __shared__ PagedPlace places[kRowsPerCta];
    pdl_wait();
    uint4 x[U][P], next[U][P];
    auto load = [&](int v0, uint4 (&to)[U][P]) {
#pragma unroll
        for (int u = 0; u < U; ++u)
        {
            const int i = v0 + (u * kRowWarps + warp) * VPW + sub;
            if (i >= nv) continue;
            const PagedVector v = paged_vector(a, i);
            const RT* const p = paged_row_at<const RT>(a, v, r0) + d;
#pragma unroll
            for (int c = 0; c < P; ++c) to[u][c] = __ldg(reinterpret_cast<const uint4*>(p + c * (D / P)));
        }
    };
    load(0, next);   // ahead of the look-ups: the values do not depend on them
    paged_places(a.c, a.b, r0, n_rows, places);
    for (int v0 = 0; v0 < nv; v0 += STEP)
    {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < P; ++c) x[u][c] = next[u][c];
        if (v0 + STEP < nv) load(v0 + STEP, next);
#pragma unroll
        for (int u = 0; u < U; ++u)
        {
            const int i = v0 + (u * kRowWarps + warp) * VPW + sub;
            const PagedVector v = paged_vector(a, min(i, nv - 1));
            const PagedPlace o = places[v.row];
            const bool live = i < nv && o.off >= 0;
            const long long at = o.off + static_cast<long long>(v.head) * a.page_head_stride + d;
            void* const pool = v.isv ? a.c.v : a.c.k;
            auto piece = [&](int c, float (&f)[E]) {   // as fp32
                const uint32_t w4[4] = {x[u][c].x, x[u][c].y, x[u][c].z, x[u][c].w};
#pragma unroll
                for (int e = 0; e < E; ++e)
                    f[e] = E == 4 ? __uint_as_float(w4[e]) : __uint_as_float((e & 1) ? w4[e >> 1] & 0xFFFF0000u : w4[e >> 1] << 16);
            };
            if constexpr (kCodes<CT>)
            {
                // The largest magnitude by its bits: an infinity or a NaN comes out on top.
                uint32_t m = 0;
#pragma unroll
                for (int c = 0; c < P; ++c)
                {
                    const uint32_t w4[4] = {x[u][c].x, x[u][c].y, x[u][c].z, x[u][c].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if constexpr (E == 8) m = __vmaxu2(m, w4[e] & 0x7fff7fffu);   // two bf16 to a word
                        else m = max(m, w4[e] & 0x7fffffffu);
                }
                if constexpr (E == 8) m = max(m << 16, m & 0x7fff0000u);
#pragma unroll
                for (int w = LPV / 2; w > 0; w >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, w));
                const bool finite = m < 0x7f800000u;
                const float scale = finite ? code_scale<CT>(__uint_as_float(m)) : __int_as_float(0x7fffffff);
                const float inv = __fdividef(1.f, scale);   // (scale < 2^126; off by 2 ulp, which quant4 allows for)
                if (live)
                {
                    uint8_t* const p = static_cast<uint8_t*>(pool) + at;
#pragma unroll
                    for (int c = 0; c < P; ++c)
                    {
                        float f[E];
                        piece(c, f);
                        uint32_t w[E / 4];
#pragma unroll
                        for (int y = 0; y < E / 4; ++y) w[y] = finite ? quant4<CT>(f + 4 * y, scale, inv) : 0u;
                        if constexpr (E == 8) *reinterpret_cast<uint2*>(p + c * (D / P)) = make_uint2(w[0], w[1]);
                        else *reinterpret_cast<uint32_t*>(p + c * (D / P)) = w[0];
                    }
                    if (lane % LPV == 0) (v.isv ? a.c.v_scale : a.c.k_scale)[o.s_off + static_cast<long long>(v.head) * a.scale_head_stride] = scale;
                }
            }
            else
            {
                if (live)
#pragma unroll
                    for (int c = 0; c < P; ++c)
                    {
                        float f[E];
                        piece(c, f);
                        store_row<CT, E>(pool, at + c * (D / P), f);
                    }
            }
        }
    }
}

template <typename RT, typename CT, int D>
__global__ void __launch_bounds__(kRowWarps * 32) paged_read_kernel(const PagedRowArgs a)
{
    constexpr int E = 16 / static_cast<int>(sizeof(RT));
    constexpr int P = 2;                                      // pieces per lane, as in the write
    constexpr int LPV = D / (E * P);
    constexpr int VPW = 32 / LPV;
    constexpr int U = E * sizeof(CT) > 16 ? 2 : 4;
    constexpr int STEP = U * kRowWarps * VPW;
    constexpr int W = E * static_cast<int>(sizeof(CT)) / 4;   // words of a piece in the cache
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r0 = blockIdx.x * a.per_cta, n_rows = min(a.per_cta, a.b.rows - r0);
    const int nv = n_rows * 2 * a.c.kv_heads, sub = lane / LPV, d = (lane % LPV) * E;
    __shared__ PagedPlace places[kRowsPerCta];
    pdl_wait();
    paged_places(a.c, a.b, r0, n_rows, places);
    for (int v0 = 0; v0 < nv; v0 += STEP)
    {
        uint32_t x[U][P][W];
        float scale[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
        {
            const int i = v0 + (u * kRowWarps + warp) * VPW + sub;
            if (i >= nv) continue;
            const PagedVector v = paged_vector(a, i);
            const PagedPlace o = places[v.row];
            if (o.off < 0) continue;
            const CT* const p = static_cast<const CT*>(v.isv ? a.c.v : a.c.k) + o.off + static_cast<long long>(v.head) * a.page_head_stride + d;
#pragma unroll
            for (int c = 0; c < P; ++c)
            {
                const CT* const pc = p + c * (D / P);
                if constexpr (W == 1) x[u][c][0] = __ldg(reinterpret_cast<const uint32_t*>(pc));
                else if constexpr (W == 2)
                {
                    const uint2 y = __ldg(reinterpret_cast<const uint2*>(pc));
                    x[u][c][0] = y.x; x[u][c][1] = y.y;
                }
                else
#pragma unroll
                    for (int w = 0; w < W; w += 4)
                    {
                        const uint4 y = __ldg(reinterpret_cast<const uint4*>(pc) + w / 4);
                        x[u][c][w] = y.x; x[u][c][w + 1] = y.y; x[u][c][w + 2] = y.z; x[u][c][w + 3] = y.w;
                    }
            }
            if constexpr (kCodes<CT>) scale[u] = __ldg((v.isv ? a.c.v_scale : a.c.k_scale) + o.s_off + static_cast<long long>(v.head) * a.scale_head_stride);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
        {
            const int i = v0 + (u * kRowWarps + warp) * VPW + sub;
            if (i >= nv) continue;
            const PagedVector v = paged_vector(a, i);
            if (places[v.row].off < 0) continue;
            RT* const to = paged_row_at<RT>(a, v, r0);
#pragma unroll
            for (int c = 0; c < P; ++c)
            {
                float f[E];
#pragma unroll
                for (int e = 0; e < E; ++e)
                {
                    if constexpr (sizeof(CT) == 4) f[e] = __uint_as_float(x[u][c][e]);
                    else if constexpr (sizeof(CT) == 2) f[e] = __uint_as_float((e & 1) ? x[u][c][e >> 1] & 0xFFFF0000u : x[u][c][e >> 1] << 16);
                    else if (e % 4 == 0) decode4<CT>(x[u][c][e / 4], f + e);
                }
                if constexpr (kCodes<CT>)
#pragma unroll
                    for (int e = 0; e < E; ++e) f[e] *= scale[u];
                store_row<RT, E>(to, d + c * (D / P), f);
            }
        }
    }
}

}  // namespace hy
