// Attention weights added up for every position of the paged cache:
//   w[j] (+)= sum over a sequence's rows i that see j, and the query heads of a KV
//   head, of exp(scale q_i k_j - lse_i),
// lse_i being the logarithm of the row's sum that its attention left. The positions
// of the rows themselves start anew (w is set there, elsewhere added to).
//
// With lse given, nothing has to be known about other keys: whoever has a
// key's scores for all rows has its sum. So the keys are split over the warps, each key
// belongs to one warp, which reads it once, and no two meet: no atomics, no second
// pass, the same bits every time.
//
// Products are taken transposed, S^T[key x column] = K Q^T (a column is a (row, head of the
// group) pair), so that a key's scores lie in one lane group. Keys go from
// memory to registers as the matrix fragments they are needed as: which dimensions a lane
// takes is free as long as q agrees, so a lane takes 16-byte pieces of its rows, and shared memory
// is not needed for them. Terms of fp32 numbers and f16 codes are those of hy_paged_attn.cuh.
// The argument of the exponential is taken as fma(score, scale, -lse) and then
// times log2(e): both roundings are relative to what is left, which is small where the
// weight is large.
#pragma once

#include "hy_paged_attn.cuh"

namespace hy {

struct PagedWeighArgs {
    PagedAttnArgs a;   // (out and work are unused, lse is read)
    float* weights;
    long long w_page_stride, w_head_stride, w_row_stride;
    float scale;
};

constexpr int kWeighAll = 1 << 30;   // columns of a tile: all of a sequence's
constexpr float kLog2e = 1.4426950408889634f;

// Dimension of the first of the four that lane t (of four) takes in k step ks, by the cache's type: its pieces of
// a row are the 16-byte pieces t, t + 4, ...
template <typename CT>
__device__ __forceinline__ int weigh_dim(int ks, int t)
{
    if constexpr (sizeof(CT) == 4) return 16 * ks + 4 * t;
    else if constexpr (sizeof(CT) == 2) return 32 * (ks >> 1) + 8 * t + 4 * (ks & 1);
    else return 64 * (ks >> 2) + 16 * t + 4 * (ks & 3);
}
// Bits of 2^-k, k = 14 - exponent of the largest magnitude of a query, kept within the normal numbers.
__device__ __forceinline__ uint32_t weigh_down_bits(uint32_t largest) { return (min(max(largest >> 23, 16u), 254u) - 14u) << 23; }

// Fragments of k step ks from a lane's pieces of rows g (x) and g + 8 (y), as NK terms.
template <typename CT, int NK>
__device__ __forceinline__ void weigh_key_frag(const uint4* x, const uint4* y, int ks, uint32_t (&ka)[NK][4])
{
    auto word = [](const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; };
    if constexpr (sizeof(CT) == 4)
    {
        const uint4 u = x[ks], v = y[ks];
        uint32_t p[NK];
        auto put = [&](int at, uint32_t lo, uint32_t hi) {
            split_pair<false, NK>(__uint_as_float(lo), __uint_as_float(hi), p);
#pragma unroll
            for (int n = 0; n < NK; ++n) ka[n][at] = p[n];
        };
        put(0, u.x, u.y);
        put(1, v.x, v.y);
        put(2, u.z, u.w);
        put(3, v.z, v.w);
    }
    else if constexpr (sizeof(CT) == 2)
    {
        const uint4 u = x[ks >> 1], v = y[ks >> 1];
        ka[0][0] = word(u, 2 * (ks & 1));
        ka[0][1] = word(v, 2 * (ks & 1));
        ka[0][2] = word(u, 2 * (ks & 1) + 1);
        ka[0][3] = word(v, 2 * (ks & 1) + 1);
    }
    else
    {
        const uint32_t u = word(x[ks >> 2], ks & 3), v = word(y[ks >> 2], ks & 3);
        ka[0][0] = codes_f16<CT>(u);
        ka[0][1] = codes_f16<CT>(v);
        ka[0][2] = codes_f16<CT, true>(u);
        ka[0][3] = codes_f16<CT, true>(v);
    }
}

// Row tensor offset of column c of a sequence's KV head.
__device__ __forceinline__ long long weigh_q_at(const PagedAttnArgs& a, const SplitItem& it, int c)
{
    const int row = paged_row_of(a, c);
    return (it.q.row0 + row) * a.q_row_stride + (it.head * a.group + c - row * a.group) * a.q_head_stride;
}
__device__ __forceinline__ float weigh_lse(const PagedAttnArgs& a, const SplitItem& it, int c)
{
    const int row = paged_row_of(a, c);
    return __ldg(a.lse + (it.q.row0 + row) * a.lse_row_stride + (it.head * a.group + c - row * a.group) * a.lse_head_stride);
}
__device__ __forceinline__ int weigh_pos(const PagedAttnArgs& a, const SplitItem& it, int c)
{
    return c < it.cols ? it.q.kv - it.q.n + paged_row_of(a, c) : -1;
}
// What a column has of a key, from their product; d's rounding is relative to d.
__device__ __forceinline__ float weigh_exp(float s, float fac, float lse) { return ex2(fmaf(s, fac, -lse) * kLog2e); }

// Keys of a warp's step: a key's scale in the lane that has its number, and which keys are there.
struct WeighKey {
    float scale;
    uint32_t mask;
};

// ---------------------------------------------------------------------------
// Few columns. Every warp streams its keys through a cp.async ring of its own, three steps of 4 KB ahead (with the next
// step in registers 64 tokens over 1024-8192 E4M3 keys took 103 us; they take 76, 4.3 TB/s), with q in registers. One
// token over 2048 fp32 keys: 5.9 us.
// ---------------------------------------------------------------------------
template <typename QT_, typename CT_, int D_>
struct WeighMma {
    using QT = QT_;
    using CT = CT_;
    static constexpr int D = D_, COLS = 8;
    static constexpr bool F16 = kCodes<CT>;
    static constexpr int NQ = std::is_same_v<QT, float> ? (F16 ? 2 : 3) : 1;
    static constexpr int RB = D * static_cast<int>(sizeof(CT));
    static constexpr int KEYS = RB <= 128 ? 32 : 16, HV = KEYS / 16, KS = D / 16;
    static constexpr int PIECES = RB / 64;             // of a row, a lane's
    static constexpr int RAW = HV * 2 * PIECES;        // [hv][row g, g + 8][piece]
    static constexpr int NA = 4;                       // chains of a score's leading products: short, since the tensor cores cut sums

    uint2 qf[NQ][KS];   // column g
    float lse[2], fac[2];
    int pos[2];         // of columns 2 t, 2 t + 1
    bool full;          // all columns are there

    static __device__ __forceinline__ int row_of(int lane, int i) { return 16 * (i / (2 * PIECES)) + 8 * (i / PIECES & 1) + (lane >> 2); }
    static __device__ __forceinline__ int piece_of(int lane, int i) { return (lane & 3) + 4 * (i % PIECES); }

    __device__ __forceinline__ void columns(const PagedWeighArgs& w, const SplitItem& it, int c0)
    {
        const PagedAttnArgs& a = w.a;
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        const bool there = c0 + g < it.cols;
        const long long at = weigh_q_at(a, it, min(c0 + g, it.cols - 1));
        float x[KS][4];
        uint32_t most = 0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
        {
            load_row<QT, 4>(a.q, at + weigh_dim<CT>(ks, t), x[ks]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
            {
                if (!there) x[ks][e] = 0.f;
                most = max(most, __float_as_uint(x[ks][e]) & 0x7fffffffu);
            }
        }
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const uint32_t down = F16 ? weigh_down_bits(most) : 127u << 23;
        const float up = __uint_as_float((254u << 23) - down);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
        {
            uint32_t b0[NQ], b1[NQ];
            split_pair<F16, NQ>(x[ks][0] * up, x[ks][1] * up, b0);
            split_pair<F16, NQ>(x[ks][2] * up, x[ks][3] * up, b1);
#pragma unroll
            for (int j = 0; j < NQ; ++j) qf[j][ks] = make_uint2(b0[j], b1[j]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
        {
            const int c = c0 + 2 * t + e;
            pos[e] = weigh_pos(a, it, c);
            lse[e] = weigh_lse(a, it, min(c, it.cols - 1));
            fac[e] = w.scale * __uint_as_float(__shfl_sync(0xffffffffu, down, 4 * (2 * t + e)));
        }
        full = c0 + COLS <= it.cols;
    }

    // The sum of the key that has this lane's number.
    __device__ __forceinline__ float step(const PagedAttnArgs& a, const SplitItem& it, int u0, const uint4 (&raw)[RAW], const WeighKey& key)
    {
        const int lane = threadIdx.x & 31, g = lane >> 2;
        const bool whole = full && split_whole<KEYS>(a, it, u0, key.mask);
        float mine = 0.f;
#pragma unroll
        for (int hv = 0; hv < HV; ++hv)
        {
            float part[NA + (NQ > 1)][4];
#pragma unroll
            for (int n = 0; n < NA + (NQ > 1); ++n) part[n][0] = part[n][1] = part[n][2] = part[n][3] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
            {
                uint32_t ka[1][4];
                weigh_key_frag<CT, 1>(raw + hv * 2 * PIECES, raw + hv * 2 * PIECES + PIECES, ks, ka);
#pragma unroll
                for (int j = NQ - 1; j > 0; --j) mma16816<F16>(part[NA], ka[0], qf[j][ks].x, qf[j][ks].y);
                mma16816<F16>(part[ks % NA], ka[0], qf[0][ks].x, qf[0][ks].y);
            }
#pragma unroll
            for (int r = 0; r < 2; ++r)
            {
                const int k = 16 * hv + 8 * r + g;
                const float kf = F16 ? __shfl_sync(0xffffffffu, key.scale, k) : 1.f;
                const int j = split_key(it, u0 + k);
                const bool there = (key.mask >> k) & 1u;
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 2; ++e)
                {
                    float s = (part[0][2 * r + e] + part[1][2 * r + e]) + (part[2][2 * r + e] + part[3][2 * r + e]);
                    if constexpr (NQ > 1) s = part[NA][2 * r + e] + s;
                    const float p = weigh_exp(F16 ? s * kf : s, fac[e], lse[e]);
                    sum += (whole || (there && paged_sees(a, pos[e], j))) ? p : 0.f;
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                const float of_key = __shfl_sync(0xffffffffu, sum, (lane & 7) * 4);
                if ((lane >> 3) == 2 * hv + r) mine = of_key;
            }
        }
        return mine;
    }
};

// fp32 caches and up to 4 columns: plain multiply-adds; eight lanes share a key, as in FmaEngine.
template <typename QT_, int D_, int NC>
struct WeighFma {
    using QT = QT_;
    using CT = float;
    static constexpr int D = D_, COLS = NC;
    static constexpr bool F16 = false;
    static constexpr int RB = D * 4, KEYS = 4096 / RB, P = D / 32, KK = KEYS / 4, RAW = KK * P;

    float4 q[NC][P];
    float lse[NC], scale;
    int pos[NC];
    bool full;

    static __device__ __forceinline__ int row_of(int lane, int i) { return 4 * (i / P) + (lane >> 3); }
    static __device__ __forceinline__ int piece_of(int lane, int i) { return (lane & 7) + 8 * (i % P); }

    __device__ __forceinline__ void columns(const PagedWeighArgs& w, const SplitItem& it, int c0)
    {
        const int dl = threadIdx.x & 7;
#pragma unroll
        for (int c = 0; c < NC; ++c)
        {
            const int cc = min(c0 + c, it.cols - 1);
            const long long at = weigh_q_at(w.a, it, cc);
#pragma unroll
            for (int p = 0; p < P; ++p)
            {
                float x[4];
                load_row<QT, 4>(w.a.q, at + (dl + 8 * p) * 4, x);
                q[c][p] = make_float4(x[0], x[1], x[2], x[3]);
            }
            pos[c] = weigh_pos(w.a, it, c0 + c);
            lse[c] = weigh_lse(w.a, it, cc);
        }
        scale = w.scale;
        full = c0 + COLS <= it.cols;
    }

    __device__ __forceinline__ float step(const PagedAttnArgs& a, const SplitItem& it, int u0, const uint4 (&raw)[RAW], const WeighKey& key)
    {
        const int lane = threadIdx.x & 31, kg = lane >> 3;
        float s[KK][NC];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int c = 0; c < NC; ++c)
            {
                s[kk][c] = 0.f;
#pragma unroll
                for (int p = 0; p < P; ++p)
                {
                    const uint4& x = raw[kk * P + p];
                    s[kk][c] += dot4(q[c][p], make_float4(__uint_as_float(x.x), __uint_as_float(x.y), __uint_as_float(x.z), __uint_as_float(x.w)));
                }
            }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1)
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int c = 0; c < NC; ++c) s[kk][c] += __shfl_xor_sync(0xffffffffu, s[kk][c], o);
        const bool whole = full && split_whole<KEYS>(a, it, u0, key.mask);
        float mine = 0.f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
        {
            const int k = 4 * kk + kg, j = split_key(it, u0 + k);
            const bool there = (key.mask >> k) & 1u;
            float sum = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c)
            {
                const float p = weigh_exp(s[kk][c], scale, lse[c]);
                sum += (whole || (there && paged_sees(a, pos[c], j))) ? p : 0.f;
            }
            const float of_key = __shfl_sync(0xffffffffu, sum, (lane & 3) * 8);
            if ((lane >> 2) == kk) mine = of_key;
        }
        return mine;
    }
};

constexpr int kWeighCtas = 3;   // per SM
constexpr int kWeighRing = 4;   // steps of a warp's ring
// A step in the ring: the lanes' pieces, then by key where its weight is, what it has (0 for a new row's), its scale; the mask.
template <typename E>
struct WeighShape {
    static constexpr int AT = E::RAW * 512, OLD = AT + 256, SCALE = OLD + 128, MASK = SCALE + 128, STAGE = MASK + 16;
    static constexpr int SMEM = kSplitWarps * kWeighRing * STAGE;
    static_assert(SMEM * kWeighCtas <= 224 * 1024, "shared memory");
};

template <typename E>
__global__ void __launch_bounds__(kSplitThreads, kWeighCtas) paged_weigh_kernel(const PagedWeighArgs w)
{
    using CT = typename E::CT;
    constexpr int KEYS = E::KEYS, TILE = kSplitWarps * KEYS, PIECE = 16 / static_cast<int>(sizeof(CT));
    using Sh = WeighShape<E>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ long long scan[kSplitWarps + 1];
    const PagedAttnArgs& a = w.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kr = lane % KEYS;
    unsigned char* const ring = smem + warp * kWeighRing * Sh::STAGE;
    const uint32_t ring_u = smem_u32(ring);
    pdl_wait();
    pdl_launch();
    const SplitStart st = split_start<kWeighAll, TILE, kSplitThreads>(a, scan);
    if (st.x0 >= st.x1) return;
    SplitItem it;
    it.seq = st.seq;
    it.tile = 0;
    if (!paged_seq(a.b, it.seq, a.c.page_size, nullptr, it.q)) return;   // (the arrays changed under the call)
    it.w = paged_span(a, it.q, 0, kWeighAll);
    it.tiles = split_tiles<TILE>(it.w.n);
    const int units = (it.tiles + st.unit - 1) / st.unit;
    it.head = split_div(st.in_seq, units);
    int tile0 = static_cast<int>(st.in_seq - static_cast<long long>(it.head) * units) * st.unit;
    long long left = (st.x1 - st.x0) * st.unit;
    E eng;
    while (true)
    {
        const int tile1 = static_cast<int>(min(static_cast<long long>(it.tiles), tile0 + left)), n_tiles = tile1 - tile0;
        it.cols = it.q.n * a.group;
        const int* const table = a.b.table + it.seq * a.b.table_stride;
        for (int c0 = 0; c0 < it.cols; c0 += E::COLS)
        {
            // Page and row in it of this lane's key of a tile (looked up a step ahead of the load).
            auto look_up = [&](int i, int& pg, int& row) {
                const int u = (tile0 + i) * TILE + warp * KEYS + kr;
                if (i >= n_tiles || u >= it.w.n) return;
                const int j = split_key(it, u), x = a.page_shift >= 0 ? j >> a.page_shift : j / a.c.page_size;
                row = j - x * a.c.page_size;
                pg = __ldg(table + x);
            };
            auto load = [&](int i, int pg, int row) {
                if (i < n_tiles)
                {
                    const int u = (tile0 + i) * TILE + warp * KEYS + kr, slot = i % kWeighRing;
                    const bool live = u < it.w.n, ok = live && pg >= 0 && pg < a.c.num_pages;
                    if (live && !ok) paged_status(a.c.status, kPagedBadPage);
                    uint32_t mask = __ballot_sync(0xffffffffu, ok);
                    if constexpr (KEYS < 32) mask &= (1u << KEYS) - 1u;
                    const long long off = ok ? pg * a.c.page_stride + row * a.c.row_stride + it.head * a.c.head_stride : 0;
                    const uint32_t to = ring_u + slot * Sh::STAGE;
#pragma unroll
                    for (int x = 0; x < E::RAW; ++x)
                    {
                        const int r = E::row_of(lane, x);
                        const long long o = __shfl_sync(0xffffffffu, off, r) + E::piece_of(lane, x) * PIECE;
                        cp_async16_zfill(to + x * 512 + lane * 16, static_cast<const CT*>(a.c.k) + o, (mask >> r) & 1u);
                    }
                    const long long at = ok ? pg * w.w_page_stride + row * w.w_row_stride + it.head * w.w_head_stride : 0;
                    // (the first columns' pass sets the weights of new rows)
                    cp_async4_zfill(to + Sh::OLD + lane * 4, w.weights + at, ok && !(c0 == 0 && split_key(it, u) >= it.q.kv - it.q.n));
                    if constexpr (E::F16)
                        cp_async4_zfill(to + Sh::SCALE + lane * 4, a.c.k_scale + (ok ? pg * a.c.s_page_stride + row * a.c.s_row_stride + it.head * a.c.s_head_stride : 0), ok);
                    reinterpret_cast<volatile long long*>(ring + slot * Sh::STAGE + Sh::AT)[lane] = at;
                    if (lane == 0) *reinterpret_cast<volatile uint32_t*>(ring + slot * Sh::STAGE + Sh::MASK) = mask;
                }
                cp_commit();
            };
            int pg[kWeighRing], row[kWeighRing];
#pragma unroll
            for (int i = 0; i < kWeighRing; ++i)
            {
                pg[i] = -1;
                row[i] = 0;
                look_up(i, pg[i], row[i]);
            }
#pragma unroll
            for (int i = 0; i < kWeighRing - 1; ++i) load(i, pg[i], row[i]);
            int pg1 = pg[kWeighRing - 1], row1 = row[kWeighRing - 1];
            eng.columns(w, it, c0);
            for (int i = 0; i < n_tiles; ++i)
            {
                cp_wait<kWeighRing - 2>();
                __syncwarp();
                load(i + kWeighRing - 1, pg1, row1);
                look_up(i + kWeighRing, pg1, row1);
                const int u0 = (tile0 + i) * TILE + warp * KEYS;
                if (u0 >= it.w.n) continue;   // (uniform)
                const unsigned char* const from = ring + i % kWeighRing * Sh::STAGE;
                uint4 raw[E::RAW];
#pragma unroll
                for (int x = 0; x < E::RAW; ++x) raw[x] = *reinterpret_cast<const uint4*>(from + x * 512 + lane * 16);
                WeighKey key;
                key.mask = *reinterpret_cast<const volatile uint32_t*>(from + Sh::MASK);
                key.scale = E::F16 ? reinterpret_cast<const volatile float*>(from + Sh::SCALE)[lane] : 0.f;
                const float sum = eng.step(a, it, u0, raw, key);
                if (lane < KEYS && ((key.mask >> lane) & 1u))
                    w.weights[reinterpret_cast<const volatile long long*>(from + Sh::AT)[lane]] =
                        reinterpret_cast<const volatile float*>(from + Sh::OLD)[lane] + sum;
            }
            cp_wait<0>();
            __syncwarp();   // the ring was read
        }
        left -= n_tiles;
        if (left <= 0 || st.unit > 1) break;
        tile0 = 0;
        if (++it.head == a.c.kv_heads)
        {
            it.head = 0;
            do
            {
                ++it.seq;
            } while (it.seq < a.b.num_seqs && (!paged_seq(a.b, it.seq, a.c.page_size, nullptr, it.q) || it.q.n == 0));
            if (it.seq >= a.b.num_seqs) break;   // (the arrays changed under the call)
            it.w = paged_span(a, it.q, 0, kWeighAll);
            it.tiles = split_tiles<TILE>(it.w.n);
        }
    }
}

// ---------------------------------------------------------------------------
// Many columns: the keys stay, q streams. Each of 8 warps holds 16 or 32 keys as fragments; the
// CTA turns q into fragments in shared memory, 32 columns at a time, the next ones' loads in flight meanwhile. mma.sync
// bounds it: 4 x ~1012 bf16 rows over 6000-8192 bf16 keys took 945 us here (163 in hy_paged_weigh_chunk.cuh, which takes
// what it can); fp32 rows multiply 2 or 3 times as often, fp32 keys and rows 6 times.
// ---------------------------------------------------------------------------
constexpr int kWeighWideWarps = 8;
constexpr int kWeighWideCols = 32;

template <typename QT_, typename CT_, int D_>
struct WeighWide {
    using QT = QT_;
    using CT = CT_;
    static constexpr int D = D_, COLS = kWeighWideCols, NT = COLS / 8;
    static constexpr bool F16 = kCodes<CT>;
    static constexpr int NQ = std::is_same_v<QT, float> ? (F16 ? 2 : 3) : 1;
    static constexpr int NK = std::is_same_v<CT, float> ? 3 : 1;
    static constexpr int RB = D * static_cast<int>(sizeof(CT)), KS = D / 16, PIECES = RB / 64;
    // Keys of a warp, in 16s: 32 over 8-bit caches (4 x ~1012 fp32 rows over 6000-8192 E4M3 keys: 1.0 ms, 1.5 with 16; 2 x 350
    // rows and keys 59 us, 44 with 16), 16 over others (BF16: 1.68 ms, 1.83 with 32; 48 us, 98 with 32).
    static constexpr int HV = F16 ? 2 : 1, KEYS = 16 * HV, TILE = kWeighWideWarps * KEYS;
    static constexpr int FRAGS = NQ * KS * NT * 32;                       // uint2s of a tile of columns
    static constexpr int SMEM = 2 * (FRAGS * 8 + 3 * COLS * 4);           // two tiles: fragments, lse, factor, position
    static constexpr int QI = KS / 2;                                     // fragments that a thread makes
};

template <typename E>
__global__ void __launch_bounds__(kWeighWideWarps * 32, 1) paged_weigh_wide_kernel(const PagedWeighArgs w)
{
    using CT = typename E::CT;
    using QT = typename E::QT;
    constexpr int KEYS = E::KEYS, TILE = E::TILE, KS = E::KS, NT = E::NT, NQ = E::NQ, NK = E::NK, HV = E::HV, PIECES = E::PIECES;
    constexpr int COLS = E::COLS, PIECE = 16 / static_cast<int>(sizeof(CT)), NA = 2;
    constexpr bool F16 = E::F16;
    extern __shared__ __align__(128) unsigned char smem[];
    uint2* const frags = reinterpret_cast<uint2*>(smem);                          // [2][term][ks][nt][lane]
    float* const lse_s = reinterpret_cast<float*>(smem + 2 * E::FRAGS * 8);       // [2][COLS]
    float* const fac_s = lse_s + 2 * COLS;
    int* const pos_s = reinterpret_cast<int*>(fac_s + 2 * COLS);
    __shared__ long long scan[kWeighWideWarps + 1];
    const PagedAttnArgs& a = w.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, kr = lane % KEYS;
    pdl_wait();
    pdl_launch();
    const SplitStart st = split_start<kWeighAll, TILE, kWeighWideWarps * 32>(a, scan);
    if (st.x0 >= st.x1) return;
    SplitItem it;
    it.seq = st.seq;
    it.tile = 0;
    if (!paged_seq(a.b, it.seq, a.c.page_size, nullptr, it.q)) return;   // (the arrays changed under the call)
    it.w = paged_span(a, it.q, 0, kWeighAll);
    it.tiles = split_tiles<TILE>(it.w.n);
    const int units = (it.tiles + st.unit - 1) / st.unit;
    it.head = split_div(st.in_seq, units);
    int tile = static_cast<int>(st.in_seq - static_cast<long long>(it.head) * units) * st.unit;
    int buf = 0;
    for (long long left = (st.x1 - st.x0) * st.unit; left > 0; --left)
    {
        it.cols = it.q.n * a.group;
        // ---- the tile's keys ----
        const int u0 = tile * TILE + warp * KEYS, u = u0 + kr;
        bool ok = false;
        long long off = 0, at = 0;
        float kf_mine = 0.f;
        int j_mine = 0;
        if (u < it.w.n)
        {
            j_mine = split_key(it, u);
            const int x = a.page_shift >= 0 ? j_mine >> a.page_shift : j_mine / a.c.page_size, row = j_mine - x * a.c.page_size;
            const int pg = __ldg(a.b.table + it.seq * a.b.table_stride + x);
            ok = pg >= 0 && pg < a.c.num_pages;
            if (!ok) paged_status(a.c.status, kPagedBadPage);
            else
            {
                off = pg * a.c.page_stride + row * a.c.row_stride + it.head * a.c.head_stride;
                at = pg * w.w_page_stride + row * w.w_row_stride + it.head * w.w_head_stride;
                if constexpr (F16) kf_mine = __ldg(a.c.k_scale + pg * a.c.s_page_stride + row * a.c.s_row_stride + it.head * a.c.s_head_stride);
            }
        }
        uint32_t mask = __ballot_sync(0xffffffffu, ok);
        if constexpr (KEYS < 32) mask &= (1u << KEYS) - 1u;
        uint32_t ka[HV][KS][NK][4];
#pragma unroll
        for (int hv = 0; hv < HV; ++hv)
        {
            uint4 raw[2][PIECES];
#pragma unroll
            for (int r = 0; r < 2; ++r)
            {
                const int k = 16 * hv + 8 * r + g;
                const CT* const p = static_cast<const CT*>(a.c.k) + __shfl_sync(0xffffffffu, off, k);
#pragma unroll
                for (int x = 0; x < PIECES; ++x)
                    raw[r][x] = (mask >> k) & 1u ? __ldg(reinterpret_cast<const uint4*>(p + (t + 4 * x) * PIECE)) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) weigh_key_frag<CT, NK>(raw[0], raw[1], ks, ka[hv][ks]);
        }
        int key[HV][2];
        float kf[HV][2], sum[HV][2];
#pragma unroll
        for (int hv = 0; hv < HV; ++hv)
#pragma unroll
            for (int r = 0; r < 2; ++r)
            {
                key[hv][r] = __shfl_sync(0xffffffffu, j_mine, 16 * hv + 8 * r + g);
                kf[hv][r] = __shfl_sync(0xffffffffu, kf_mine, 16 * hv + 8 * r + g);
                sum[hv][r] = 0.f;
            }

        // ---- the columns that see any of the CTA's keys ----
        const int p_0 = it.q.kv - it.q.n, u_last = min((tile + 1) * TILE, it.w.n) - 1;
        const int j_first = split_key(it, tile * TILE), j_last = split_key(it, max(u_last, 0));
        int row_a = max(0, -p_0), row_b = it.q.n;
        if (a.causal) row_a = max(row_a, j_first - p_0);
        if (a.window > 0 && j_first >= a.sinks)   // (rows from j + window on do not see j)
            row_b = static_cast<int>(min(static_cast<long long>(row_b), static_cast<long long>(j_last) + a.window - p_0));
        const int c_begin = row_a * a.group / COLS * COLS, c_end = u_last < tile * TILE ? 0 : row_b * a.group;
        // A thread makes the fragments of one column: 4 columns to a warp, eight lanes to a column.
        const int qc = warp * 4 + (lane >> 3), qs = lane & 7, qt = qs & 3;
        float x[E::QI][4], x_lse = 0.f;
        auto fetch = [&](int c0) {
            const int c = min(c0 + qc, it.cols - 1);
            const long long o = weigh_q_at(a, it, c);
#pragma unroll
            for (int i = 0; i < E::QI; ++i) load_row<QT, 4>(a.q, o + weigh_dim<CT>(2 * i + (qs >> 2), qt), x[i]);
            x_lse = weigh_lse(a, it, c);
        };
        if (c_begin < c_end) fetch(c_begin);
        for (int c0 = c_begin; c0 < c_end; c0 += COLS, buf ^= 1)
        {
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < E::QI; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                {
                    if (c0 + qc >= it.cols) x[i][e] = 0.f;
                    most = max(most, __float_as_uint(x[i][e]) & 0x7fffffffu);
                }
            uint32_t down = 127u << 23;
            if constexpr (F16)
            {
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
                down = weigh_down_bits(most);
            }
            const float up = __uint_as_float((254u << 23) - down);
            uint2* const to = frags + buf * E::FRAGS;
#pragma unroll
            for (int i = 0; i < E::QI; ++i)
            {
                uint32_t b0[NQ], b1[NQ];
                split_pair<F16, NQ>(x[i][0] * up, x[i][1] * up, b0);
                split_pair<F16, NQ>(x[i][2] * up, x[i][3] * up, b1);
#pragma unroll
                for (int j = 0; j < NQ; ++j)
                    to[((j * KS + 2 * i + (qs >> 2)) * NT + (qc >> 3)) * 32 + (qc & 7) * 4 + qt] = make_uint2(b0[j], b1[j]);
            }
            if (qs == 0)
            {
                lse_s[buf * COLS + qc] = x_lse;
                fac_s[buf * COLS + qc] = w.scale * __uint_as_float(down);
                pos_s[buf * COLS + qc] = weigh_pos(a, it, c0 + qc);
            }
            if (c0 + COLS < c_end) fetch(c0 + COLS);
            __syncthreads();   // (the buffer after this one was last read before the barrier before this one)
            if (mask == 0) continue;
            // Every column of the tile sees every key of the warp.
            const int p_first = p_0 + paged_row_of(a, c0), p_last = p_0 + paged_row_of(a, min(c0 + COLS, it.cols) - 1);
            const int jf = split_key(it, u0), jl = split_key(it, u0 + KEYS - 1);
            const bool whole = c0 + COLS <= it.cols && mask == (KEYS == 32 ? 0xffffffffu : (1u << (KEYS & 31)) - 1u) && p_first >= 0 &&
                               (!a.causal || (jl <= p_first && (a.window == 0 || jf > p_last - a.window || jl < a.sinks)));
#pragma unroll
            for (int n0 = 0; n0 < NT; n0 += 2)
            {
                float part[NA][HV][2][4];   // the leading products, and the small terms' (apart: the tensor cores cut sums)
#pragma unroll
                for (int n = 0; n < NA; ++n)
#pragma unroll
                    for (int hv = 0; hv < HV; ++hv)
#pragma unroll
                        for (int y = 0; y < 2; ++y) part[n][hv][y][0] = part[n][hv][y][1] = part[n][hv][y][2] = part[n][hv][y][3] = 0.f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int j = NQ - 1; j >= 0; --j)
#pragma unroll
                        for (int y = 0; y < 2; ++y)
                        {
                            const uint2 b = to[((j * KS + ks) * NT + n0 + y) * 32 + lane];
#pragma unroll
                            for (int n = NK - 1; n >= 0; --n)
#pragma unroll
                                for (int hv = 0; hv < HV; ++hv)
                                    if (n + j <= 2) mma16816<F16>(part[NQ * NK == 1 ? ks % NA : (n + j > 0 ? 1 : 0)][hv][y], ka[hv][ks][n], b.x, b.y);
                        }
#pragma unroll
                for (int y = 0; y < 2; ++y)
                {
                    const int c = buf * COLS + (n0 + y) * 8 + 2 * t;
                    const float2 lse = *reinterpret_cast<const float2*>(lse_s + c), fac = *reinterpret_cast<const float2*>(fac_s + c);
                    const int2 pos = *reinterpret_cast<const int2*>(pos_s + c);
#pragma unroll
                    for (int hv = 0; hv < HV; ++hv)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                        {
                            const int r = e >> 1;
                            float s = part[1][hv][y][e] + part[0][hv][y][e];
                            if constexpr (F16) s *= kf[hv][r];
                            const float p = weigh_exp(s, e & 1 ? fac.y : fac.x, e & 1 ? lse.y : lse.x);
                            const bool seen = whole || (((mask >> (16 * hv + 8 * r + g)) & 1u) && paged_sees(a, e & 1 ? pos.y : pos.x, key[hv][r]));
                            sum[hv][r] += seen ? p : 0.f;
                        }
                }
            }
        }

        // ---- a key's sum to the lane that has its number ----
        float mine = 0.f;
#pragma unroll
        for (int hv = 0; hv < HV; ++hv)
#pragma unroll
            for (int r = 0; r < 2; ++r)
            {
                float s = sum[hv][r];
                s += __shfl_xor_sync(0xffffffffu, s, 1);
                s += __shfl_xor_sync(0xffffffffu, s, 2);
                const float of_key = __shfl_sync(0xffffffffu, s, (lane & 7) * 4);
                if ((lane >> 3) == 2 * hv + r) mine = of_key;
            }
        if (ok && lane < KEYS) w.weights[at] = (j_mine >= p_0 ? 0.f : w.weights[at]) + mine;

        if (++tile == it.tiles)
        {
            if (st.unit > 1) break;
            tile = 0;
            if (++it.head == a.c.kv_heads)
            {
                it.head = 0;
                do
                {
                    ++it.seq;
                } while (it.seq < a.b.num_seqs && (!paged_seq(a.b, it.seq, a.c.page_size, nullptr, it.q) || it.q.n == 0));
                if (it.seq >= a.b.num_seqs) break;   // (the arrays changed under the call)
                it.w = paged_span(a, it.q, 0, kWeighAll);
                it.tiles = split_tiles<TILE>(it.w.n);
            }
        }
    }
}

}  // namespace hy
