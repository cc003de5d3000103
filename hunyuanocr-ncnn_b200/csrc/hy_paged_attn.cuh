// Attention of a batch's rows over the paged cache.
//
// out = softmax(scale * q k^T) v over the positions that a row sees, in one
// pass over the keys: a running maximum m, the sum l of 2^(s - m) and the sum
// of 2^(s - m) v are kept in fp32 and rescaled when m grows (s in units of
// log 2). Parts of the keys are joined by the same rescaling.
//
// What a tile of rows sees is one run of "virtual" positions: the sinks before
// its window, then the window's positions up to the last row's; neither the
// gap between them nor what lies behind the last row is ever loaded.
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
    int page_shift;       // log2(page_size), or -1
    float scale_log2;     // scale * log2(e)
    void* work;           // workspace
};

// The keys that the columns [c0, c0 + cols) of a sequence see. A column is a
// (row, head of the group) pair: column c is row c / group.
struct PagedSpan {
    int p_first, p_last;   // positions of the first and last row
    int sinks, lo, n;      // virtual position u < sinks: u, else lo + u - sinks; n of them
};
__device__ __forceinline__ PagedSpan paged_span(const PagedAttnArgs& a, const PagedSeq& s, int c0, int cols)
{
    PagedSpan o;
    const int last = min(s.n * a.group, c0 + cols) - 1;
    o.p_first = s.kv - s.n + c0 / a.group;
    o.p_last = s.kv - s.n + last / a.group;
    const int hi = o.p_last < 0 ? 0 : a.causal ? o.p_last + 1 : s.kv;
    o.lo = (a.window > 0) ? min(hi, max(0, o.p_first - a.window + 1)) : 0;
    o.sinks = min(o.lo, a.sinks);
    o.n = o.sinks + hi - o.lo;
    return o;
}
__device__ __forceinline__ bool paged_sees(const PagedAttnArgs& a, int p, int j)
{
    if (p < 0) return false;
    if (!a.causal) return true;
    return j <= p && (a.window == 0 || p - j < a.window || j < a.sinks);
}

// ---------------------------------------------------------------------------
// Warp-level tensor core products.
// ---------------------------------------------------------------------------
// c[16 x 8] += a[16 x 16] b[16 x 8]; lane (g = lane / 4, t = lane % 4) holds
// a0: (row g, cols 2t, 2t+1), a1: row g + 8, a2: cols + 8, a3: both; b0: (rows
// 2t, 2t+1, col g), b1: rows + 8; c0, c1: (row g, cols 2t, 2t+1), c2, c3: row g + 8.
template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr)
{
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float lds_f32(uint32_t addr)
{
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool pred)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(pred ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4_zfill(uint32_t dst, const void* src, bool pred)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(pred ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi)
{
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// A pair of fp32 as T 16-bit terms (packed: lo in the low half) that add up to it.
//   bf16, 1 term: rounded. bf16, 3 terms: the leading 8 bits of the significand,
//   the next 8, the last 8 (cut, not rounded: exact, and never above the value).
//   f16, 1 or 2 terms: rounded, then the rounded remainder (22 bits and more).
template <bool F16, int T>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&o)[T])
{
    if constexpr (F16)
    {
        o[0] = pack_f16(x, y);
        if constexpr (T == 2)
        {
            const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&o[0]));
            o[1] = pack_f16(x - h.x, y - h.y);
        }
    }
    else if constexpr (T == 1)
    {
        o[0] = pack_bf16(x, y);
    }
    else
    {
#pragma unroll
        for (int i = 0; i < T; ++i)
        {
            o[i] = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
            x -= __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
            y -= __uint_as_float(__float_as_uint(y) & 0xFFFF0000u);
        }
    }
}

// Two 8-bit codes as a pair of f16 (exact for both types). x holds them in its low 16 bits.
template <typename CT>
__device__ __forceinline__ uint32_t codes_f16(uint32_t x)
{
    if constexpr (std::is_same_v<CT, E4M3>)
    {
        uint32_t y;
        asm("{.reg .b16 t, u;\n\tmov.b32 {t, u}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(y) : "r"(x));
        return y;
    }
    else
    {
        // 0x6400 | (code ^ 0x80) is 1024 + 128 + code in f16.
        const uint32_t y = (__byte_perm(x, 0, 0x4140) & 0x00ff00ffu) ^ 0x64806480u;
        const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const __half2 z = __hsub2(*reinterpret_cast<const __half2*>(&y), bias);
        return *reinterpret_cast<const uint32_t*>(&z);
    }
}

// ---------------------------------------------------------------------------
// Few rows per sequence: the keys are split over the GPU.
//
// The work is the list of (sequence, tile of 8 NT columns, KV head) items, each
// of ceil(keys / TILE) tiles (at least one), T in all; CTA i of G takes the next
// ceil(T / G) tiles of the whole list, whatever items they belong to, so every CTA
// streams the same number of keys however ragged the lengths are. Memory bounds it
// (a key is used by the group's heads only), so all that matters is that loads
// never pause: every warp owns a quarter of a tile's keys and a cp.async ring of its
// own, and the warps meet only at the end of an item.
//
// The products are taken transposed, S^T[key x column] = K Q^T and O^T[dim x
// column] = V^T P^T: with the columns in the 8-wide dimension a decode step of
// two heads wastes 6 of 8 lanes instead of 14 of 16, the accumulators of
// 128 dimensions are 32 registers, and a column's softmax state lies in the same lane for
// the scores and for the output.
//
// Operands: bf16 and fp32 caches in bf16 (an fp32 number as three terms, products
// of terms i + j <= 2: exact to 2^-23), 8-bit caches in f16, where their codes and
// the query (each row times a power of two) are exact; fp32 queries take two f16
// terms there. Which dimensions a lane takes from a row is free as long as q
// agrees, so 8-bit and fp32 keys are read from shared memory in 16-byte pieces.
//
// A CTA's first and last items may be shared with its neighbours: those leave
// (m, l, sum) parts in the workspace, slot 2 i for the first item and 2 i + 1 for a
// later one, and paged_join_kernel adds up the parts of an item. The CTA that
// starts such an item leaves its description.
// ---------------------------------------------------------------------------
constexpr int kSplitWarps = 4;
constexpr int kSplitThreads = kSplitWarps * 32;
constexpr int kSplitMaxCtas = 3 * 148;   // three CTAs per SM

struct PagedJoin {   // description of an item whose parts are joined; count 0: none
    int count, first_slot, first_cta, row0, col0, cols, head, pad;
};

template <typename QT, typename CT, int D, int NT>
struct SplitShape {
    static constexpr bool F16 = kCodes<CT>;
    static constexpr int NQ = std::is_same_v<QT, float> ? (F16 ? 2 : 3) : 1;   // terms of q and of the weights
    static constexpr int NK = std::is_same_v<CT, float> ? 3 : 1;               // terms of k and v
    static constexpr int COLS = 8 * NT;
    static constexpr int RB = D * static_cast<int>(sizeof(CT));                // bytes of a row
    // Keys of a warp's step: 32 where that is 8 KB or less (the work that a step
    // costs whatever its keys - addresses, maxima, shuffles - is halved), else 16.
    static constexpr int KEYS = RB <= 128 ? 32 : 16;
    static constexpr int TILE = kSplitWarps * KEYS;
    static constexpr int STAGE = 2 * KEYS * RB;                                // a warp's keys and values
    static constexpr int SCALES = F16 ? 2 * KEYS * 4 : 0;
    static constexpr int QB = (D / 16) * NT * NQ * 256;
    static constexpr int FIX = QB + 2 * COLS * 4 + kSplitWarps * COLS * 8 + 64;
    static constexpr int fit(int kb, int most)
    {
        const int n = (kb * 1024 - FIX) / (kSplitWarps * (STAGE + SCALES + 16));
        return n < most ? n : most;
    }
    static constexpr int OCC = (NT == 1 && fit(74, 4) >= 2) ? 3 : fit(112, 4) >= 2 ? 2 : 1;
    static constexpr int S = OCC == 3 ? fit(74, 4) : OCC == 2 ? fit(112, 4) : fit(224, 4);
    static constexpr int RING = kSplitWarps * S * STAGE;
    static constexpr int MERGE = kSplitWarps * COLS * (D + 4) * 4;   // the warps' sums, over the drained ring
    static constexpr int BODY = RING > MERGE ? RING : MERGE;
    static constexpr int SC_OFF = BODY;
    static constexpr int MASK_OFF = SC_OFF + kSplitWarps * S * SCALES;   // a bit for every key that is there
    static constexpr int Q_OFF = (MASK_OFF + kSplitWarps * S * 4 + 127) / 128 * 128;
    static constexpr int QS_OFF = Q_OFF + QB;                        // [COLS] 2^-k of a column's q
    static constexpr int ML_OFF = QS_OFF + COLS * 4;                 // [warps][COLS] (m, l)
    static constexpr int SMEM = ML_OFF + kSplitWarps * COLS * 8;
    static_assert(S >= 2 && SMEM <= 227 * 1024, "shared memory");
    static constexpr int GRID = 148 * OCC;
    static constexpr bool QREG = (D / 16) * NT * 2 * NQ <= 32;       // q stays in registers
    // Part of an item in the workspace: [COLS] (m, l), then [COLS][D].
    static constexpr int PART = COLS * (D + 2);
};

// Bytes before the parts: the descriptions.
constexpr size_t kSplitDescBytes = kSplitMaxCtas * sizeof(PagedJoin);

// Output dimension of accumulator row (m tile, half) of lane group g, by how V's fragments are read.
template <typename CT, int D>
__device__ __forceinline__ int split_dim(int mt, int half, int g)
{
    if constexpr (sizeof(CT) == 4) return 32 * (mt >> 1) + 4 * g + 2 * (mt & 1) + half;
    else if constexpr (sizeof(CT) == 2) return 16 * mt + 8 * half + g;
    else return (D / 8) * g + 2 * mt + half;
}
// Where 16-byte piece c of key row r lies in a stage (bytes), for K and for V: the
// rotations keep the lanes of each shared-memory phase on different banks.
template <typename CT, int D>
__device__ __forceinline__ int split_k_at(int r, int c)
{
    constexpr int RB = D * static_cast<int>(sizeof(CT));
    if constexpr (sizeof(CT) == 2) return r * RB + ((c ^ (r & 7)) << 4);
    else if constexpr (RB >= 128) return r * RB + ((c ^ ((r & 1) << 2)) << 4);
    else return r * RB + (c << 4);
}
template <typename CT, int D>
__device__ __forceinline__ int split_v_at(int r, int c)
{
    constexpr int RB = D * static_cast<int>(sizeof(CT));
    if constexpr (sizeof(CT) == 2) return r * RB + ((c ^ (r & 7)) << 4);
    else if constexpr (RB >= 128) return r * RB + ((c ^ (r & 6)) << 4);
    else
    {
        // 64-byte rows: even rows first, so that rows 0, 2, 4, 6 span both halves of the banks.
        const int pos = (r & ~7) | ((r & 1) << 2) | ((r & 6) >> 1);
        return pos * RB + ((c ^ (pos & 2)) << 4);
    }
}

struct SplitItem {
    PagedSeq q;
    PagedSpan w;
    int seq, tile, head, tiles;
};

template <int COLS>
__device__ __forceinline__ int split_row_tiles(const PagedAttnArgs& a, int n)
{
    return (n * a.group + COLS - 1) / COLS;
}
template <int TILE>
__device__ __forceinline__ int split_tiles(int keys) { return max(1, (keys + TILE - 1) / TILE); }

// Tiles of sequence s, all its items.
template <int COLS, int TILE>
__device__ __forceinline__ long long split_cost(const PagedAttnArgs& a, int s)
{
    PagedSeq q;
    if (s >= a.b.num_seqs || !paged_seq(a.b, s, a.c.page_size, a.c.status, q)) return 0;
    long long c = 0;
    const int rt = split_row_tiles<COLS>(a, q.n);
    for (int t = 0; t < rt; ++t) c += split_tiles<TILE>(paged_span(a, q, t * COLS, COLS).n);
    return c * a.c.kv_heads;
}

// Finds the CTA's range of tiles and the item its first tile belongs to; every
// thread returns the same. scan: shared memory for 4 + 2 long longs and 2 ints.
struct SplitStart {
    long long x0, x1, total;   // the CTA's tiles; of all
    long long in_seq;          // x0 counted from its sequence's first tile
    long long share;           // tiles per CTA
    int seq;
};
template <int COLS, int TILE>
__device__ __forceinline__ SplitStart split_start(const PagedAttnArgs& a, long long* scan)
{
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __shared__ int s_seq;
    SplitStart o;
    o.total = 0;
    const int rounds = (a.b.num_seqs + kSplitThreads - 1) / kSplitThreads;
    long long mine = 0;
    for (int r = 0; r < rounds; ++r) mine = split_cost<COLS, TILE>(a, r * kSplitThreads + tid), o.total += mine;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) o.total += __shfl_xor_sync(0xffffffffu, o.total, d);
    if (lane == 0) scan[warp] = o.total;
    __syncthreads();
    o.total = 0;
    for (int w = 0; w < kSplitWarps; ++w) o.total += scan[w];
    o.share = max(1ll, (o.total + gridDim.x - 1) / gridDim.x);
    o.x0 = min(o.total, o.share * blockIdx.x);
    o.x1 = min(o.total, o.x0 + o.share);
    o.seq = 0;
    o.in_seq = 0;
    if (o.x0 >= o.x1) return o;
    long long base = 0;
    for (int r = 0; r < rounds; ++r)
    {
        if (rounds > 1) mine = split_cost<COLS, TILE>(a, r * kSplitThreads + tid);
        long long inc = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1)
        {
            const long long v = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += v;
        }
        __syncthreads();   // scan was read
        if (lane == 31) scan[warp] = inc;
        __syncthreads();
        long long before = base;
        for (int w = 0; w < warp; ++w) before += scan[w];
        for (int w = 0; w < kSplitWarps; ++w) base += scan[w];
        const long long lo = before + inc - mine;
        if (o.x0 >= lo && o.x0 < lo + mine)
        {
            s_seq = r * kSplitThreads + tid;
            scan[4] = o.x0 - lo;
        }
        if (o.x0 < base) break;   // uniform: found in this round
    }
    __syncthreads();
    o.seq = s_seq;
    o.in_seq = scan[4];
    return o;
}

template <typename QT, typename CT, int D, int NT>
__global__ void __launch_bounds__(kSplitThreads, SplitShape<QT, CT, D, NT>::OCC) paged_split_kernel(const PagedAttnArgs a)
{
    using Sh = SplitShape<QT, CT, D, NT>;
    constexpr bool F16 = Sh::F16;
    constexpr int NQ = Sh::NQ, NK = Sh::NK, COLS = Sh::COLS, S = Sh::S, RB = Sh::RB, CPR = RB / 16;
    constexpr int KS = D / 16, MTS = D / 16, KEYS = Sh::KEYS, TILE = Sh::TILE, HV = KEYS / 16;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ long long scan[6];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_launch();
    PagedJoin* const desc = static_cast<PagedJoin*>(a.work) + blockIdx.x;
    float* const parts = reinterpret_cast<float*>(static_cast<unsigned char*>(a.work) + kSplitDescBytes);

    const SplitStart st = split_start<COLS, Sh::TILE>(a, scan);
    if (st.x0 >= st.x1)
    {
        if (tid == 0) desc->count = 0;
        return;
    }
    if (tid == 0) desc->count = 0;   // (rewritten below by the same thread)

    // The first item.
    SplitItem it;
    it.seq = st.seq;
    paged_seq(a.b, it.seq, a.c.page_size, nullptr, it.q);
    long long in = st.in_seq;
    for (it.tile = 0;; ++it.tile)
    {
        it.w = paged_span(a, it.q, it.tile * COLS, COLS);
        it.tiles = split_tiles<Sh::TILE>(it.w.n);
        if (in < static_cast<long long>(it.tiles) * a.c.kv_heads) break;
        if ((it.tile + 1) * COLS >= it.q.n * a.group) return;   // (the arrays changed under the call)
        in -= static_cast<long long>(it.tiles) * a.c.kv_heads;
    }
    it.head = static_cast<int>(in / it.tiles);
    int tile0 = static_cast<int>(in % it.tiles);

    unsigned char* const ring = smem + warp * S * Sh::STAGE;
    const uint32_t ring_u = smem_u32(ring);
    const uint32_t sc_u = smem_u32(smem + Sh::SC_OFF + warp * S * Sh::SCALES);
    volatile uint32_t* const masks = reinterpret_cast<volatile uint32_t*>(smem + Sh::MASK_OFF) + warp * S;
    uint2* const qf = reinterpret_cast<uint2*>(smem + Sh::Q_OFF);   // [term][ks][nt][lane]
    float* const qscale = reinterpret_cast<float*>(smem + Sh::QS_OFF);

    long long left = st.x1 - st.x0;
    bool first = true;
    while (true)
    {
        const int tile1 = static_cast<int>(min(static_cast<long long>(it.tiles), tile0 + left));
        const int n_tiles = tile1 - tile0;
        const int cols = min(COLS, it.q.n * a.group - it.tile * COLS);
        const int* const table = a.b.table + it.seq * a.b.table_stride;

        // ---- loads: this warp's keys of tile tile0 + i into slot i % S ----
        const int kr = lane % KEYS;
        auto key_of = [&](int u) { return u < it.w.sinks ? u : it.w.lo + u - it.w.sinks; };
        // Page and row in it of this lane's key of a tile, looked up a step ahead of the load.
        int pg_next = 0, in_next = 0;
        auto look_up = [&](int i) {
            const int u = (tile0 + i) * TILE + warp * KEYS + kr;
            if (i >= n_tiles || u >= it.w.n) return;
            const int j = key_of(u), pg = a.page_shift >= 0 ? j >> a.page_shift : j / a.c.page_size;
            in_next = j - pg * a.c.page_size;
            pg_next = __ldg(table + pg);
        };
        look_up(0);
        auto load = [&](int i) {
            if (i < n_tiles)
            {
                const int slot = i % S;
                const bool live = (tile0 + i) * TILE + warp * KEYS + kr < it.w.n;
                const bool ok = live && pg_next >= 0 && pg_next < a.c.num_pages;
                if (live && !ok) paged_status(a.c.status, kPagedBadPage);
                const long long off = ok ? pg_next * a.c.page_stride + in_next * a.c.row_stride + it.head * a.c.head_stride : 0;
                const uint32_t mask = __ballot_sync(0xffffffffu, ok);
                if (lane == 0) masks[slot] = mask;
                const uint32_t base = ring_u + slot * Sh::STAGE;
#pragma unroll
                for (int x = 0; x < KEYS * CPR / 32; ++x)
                {
                    const int idx = x * 32 + lane, r = idx / CPR, c = idx % CPR;
                    const long long o = __shfl_sync(0xffffffffu, off, r) + c * (16 / static_cast<int>(sizeof(CT)));
                    const bool pr = (mask >> r) & 1u;
                    cp_async16_zfill(base + split_k_at<CT, D>(r, c), static_cast<const CT*>(a.c.k) + o, pr);
                    cp_async16_zfill(base + KEYS * RB + split_v_at<CT, D>(r, c), static_cast<const CT*>(a.c.v) + o, pr);
                }
                if constexpr (F16)
                {
                    const long long so = ok ? pg_next * a.c.s_page_stride + in_next * a.c.s_row_stride + it.head * a.c.s_head_stride : 0;
                    const uint32_t dst = sc_u + slot * Sh::SCALES + kr * 4;
                    cp_async4_zfill(dst, a.c.k_scale + so, ok);
                    cp_async4_zfill(dst + KEYS * 4, a.c.v_scale + so, ok);
                }
                look_up(i + 1);
            }
            cp_commit();
        };
#pragma unroll
        for (int i = 0; i < S - 1; ++i) load(i);

        // ---- q as B fragments ----
        if constexpr (F16)
        {
            // A column's power of two: its largest magnitude comes to lie in [2^14, 2^15).
            for (int c = warp; c < COLS; c += kSplitWarps)
            {
                uint32_t m = 0;
                if (c < cols)
                {
                    const int cc = it.tile * COLS + c, row = it.q.row0 + cc / a.group, h = it.head * a.group + cc % a.group;
                    float x[4];
                    if (lane < D / 4) load_row<QT, 4>(a.q, row * a.q_row_stride + h * a.q_head_stride + lane * 4, x);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (lane < D / 4) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
                }
                m = __reduce_max_sync(0xffffffffu, m);
                // 2^k with k = 14 - exponent, kept within the normal numbers; not finite: 1.
                const int e = min(max(static_cast<int>(m >> 23), 16), 254);
                if (lane == 0) qscale[c] = __uint_as_float(static_cast<uint32_t>(e - 14) << 23);   // its inverse
            }
            __syncthreads();
        }
        for (int x = tid; x < KS * NT * 32; x += kSplitThreads)
        {
            const int ln = x & 31, nt = (x >> 5) % NT, ks = (x >> 5) / NT, gg = ln >> 2, tt = ln & 3;
            const int c = nt * 8 + gg;
            float v[4] = {};
            if (c < cols)
            {
                const int cc = it.tile * COLS + c, row = it.q.row0 + cc / a.group, h = it.head * a.group + cc % a.group;
                const long long o = row * a.q_row_stride + h * a.q_head_stride;
                if constexpr (sizeof(CT) == 2)
                {
                    const QT* p = static_cast<const QT*>(a.q) + o + 16 * ks + 2 * tt;
                    v[0] = to_f32<QT>(p[0]); v[1] = to_f32<QT>(p[1]); v[2] = to_f32<QT>(p[8]); v[3] = to_f32<QT>(p[9]);
                }
                else
                {
                    const int d = sizeof(CT) == 4 ? 16 * ks + 4 * tt : 64 * (ks >> 2) + 16 * tt + 4 * (ks & 3);
                    load_row<QT, 4>(a.q, o + d, v);
                }
                if constexpr (F16)
                {
                    const float up = __uint_as_float((254u << 23) - __float_as_uint(qscale[c]));   // 2^k
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] *= up;
                }
            }
            uint32_t b0[NQ], b1[NQ];
            split_pair<F16, NQ>(v[0], v[1], b0);
            split_pair<F16, NQ>(v[2], v[3], b1);
#pragma unroll
            for (int i = 0; i < NQ; ++i) qf[((i * KS + ks) * NT + nt) * 32 + ln] = make_uint2(b0[i], b1[i]);
        }
        __syncthreads();
        uint2 qreg[Sh::QREG ? NQ * KS * NT : 1];
        if constexpr (Sh::QREG)
#pragma unroll
            for (int i = 0; i < NQ * KS * NT; ++i) qreg[i] = qf[i * 32 + lane];
        auto q_frag = [&](int term, int ks, int nt) {
            const int i = (term * KS + ks) * NT + nt;
            if constexpr (Sh::QREG) return qreg[i];
            else return qf[i * 32 + lane];
        };
        // Positions and score factors of this lane's columns (2t, 2t + 1 of every n tile).
        int pos[NT][2];
        float fac[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
            {
                const int c = nt * 8 + 2 * t + e;
                pos[nt][e] = c < cols ? it.q.kv - it.q.n + (it.tile * COLS + c) / a.group : -1;
                fac[nt][e] = F16 ? a.scale_log2 * qscale[c] : a.scale_log2;
            }

        float m[NT][2], l[NT][2], acc[NT][MTS][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
        {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int i = 0; i < MTS; ++i) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
        }

        // ---- the keys ----
        for (int i = 0; i < n_tiles; ++i)
        {
            cp_wait<S - 2>();
            __syncwarp();
            load(i + S - 1);
            const int u0 = (tile0 + i) * TILE + warp * KEYS;
            if (u0 >= it.w.n) continue;   // nothing for this warp in the item's last tile
            const int slot = i % S;
            const uint32_t kb = ring_u + slot * Sh::STAGE, vb = kb + KEYS * RB;
            const uint32_t live = masks[slot];

            // Scores of the step's keys: sc[hv][nt] holds keys 16 hv + g and + 8.
            float sc[HV][NT][4];
#pragma unroll
            for (int hv = 0; hv < HV; ++hv)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) sc[hv][nt][0] = sc[hv][nt][1] = sc[hv][nt][2] = sc[hv][nt][3] = 0.f;
#pragma unroll
            for (int hv = 0; hv < HV; ++hv)
            {
                uint4 w0, w1;   // 8-bit keys: 64 dimensions of rows g and g + 8
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
                {
                    uint32_t ka[NK][4];
                    if constexpr (sizeof(CT) == 2)
                    {
                        ldmatrix4(ka[0], kb + split_k_at<CT, D>(16 * hv + (lane & 15), 2 * ks + (lane >> 4)));
                    }
                    else if constexpr (sizeof(CT) == 4)
                    {
                        const uint4 x = lds128(kb + split_k_at<CT, D>(16 * hv + g, 4 * ks + t)),
                                    y = lds128(kb + split_k_at<CT, D>(16 * hv + g + 8, 4 * ks + t));
                        uint32_t p[NK];
                        auto put = [&](int at, uint32_t lo, uint32_t hi) {
                            split_pair<false, NK>(__uint_as_float(lo), __uint_as_float(hi), p);
#pragma unroll
                            for (int n = 0; n < NK; ++n) ka[n][at] = p[n];
                        };
                        put(0, x.x, x.y);
                        put(1, y.x, y.y);
                        put(2, x.z, x.w);
                        put(3, y.z, y.w);
                    }
                    else
                    {
                        if (ks % 4 == 0)
                        {
                            w0 = lds128(kb + split_k_at<CT, D>(16 * hv + g, ks + t));
                            w1 = lds128(kb + split_k_at<CT, D>(16 * hv + g + 8, ks + t));
                        }
                        const uint32_t x = ks % 4 == 0 ? w0.x : ks % 4 == 1 ? w0.y : ks % 4 == 2 ? w0.z : w0.w;
                        const uint32_t y = ks % 4 == 0 ? w1.x : ks % 4 == 1 ? w1.y : ks % 4 == 2 ? w1.z : w1.w;
                        ka[0][0] = codes_f16<CT>(x);
                        ka[0][1] = codes_f16<CT>(y);
                        ka[0][2] = codes_f16<CT>(x >> 16);
                        ka[0][3] = codes_f16<CT>(y >> 16);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = NQ - 1; j >= 0; --j)
                        {
                            const uint2 b = q_frag(j, ks, nt);
#pragma unroll
                            for (int n = NK - 1; n >= 0; --n)
                                if (n + j <= 2) mma16816<F16>(sc[hv][nt], ka[n], b.x, b.y);
                        }
                }
            }

            // Scores in units of log 2, masks, the weights' exponents. Index [hv][r]: key 16 hv + 8 r + g.
            float vs[HV][2], ev[HV][2], kf[HV][2];
#pragma unroll
            for (int hv = 0; hv < HV; ++hv)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                {
                    kf[hv][r] = vs[hv][r] = 1.f;
                    ev[hv][r] = 0.f;
                    if constexpr (F16)
                    {
                        const uint32_t at = sc_u + slot * Sh::SCALES + (16 * hv + 8 * r + g) * 4;
                        kf[hv][r] = lds_f32(at);
                        const float v = lds_f32(at + KEYS * 4);
                        // The maximum is taken over the score plus the exponent of the value's scale, so that
                        // a weight times its scale is below 2 and fits f16 (times 2^14).
                        ev[hv][r] = static_cast<float>(min(max(static_cast<int>(__float_as_uint(v) >> 23) - 127, -100), 100));
                        vs[hv][r] = v * 16384.f;
                    }
                }
            const int j_first = key_of(u0), j_last = key_of(min(u0 + KEYS - 1, it.w.n - 1));
            const bool whole = live == (KEYS == 32 ? 0xffffffffu : 0xffffu) &&
                               (!a.causal || (j_last <= it.w.p_first &&
                                              (a.window == 0 || j_first > it.w.p_last - a.window || j_last < a.sinks))) &&
                               it.w.p_first >= 0;
            uint32_t seen = 0xffffffffu;   // bit ((hv * 2 + r) * NT + nt) * 2 + e: the column sees the key
            bool hidden = false;           // some column does not see a key that was loaded
            if (!whole)
            {
#pragma unroll
                for (int hv = 0; hv < HV; ++hv)
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                    {
                        const int in16 = 16 * hv + 8 * r + g, j = key_of(u0 + in16);
                        const bool there = (live >> in16) & 1u;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                            {
                                const bool v = there && paged_sees(a, pos[nt][e], j);
                                hidden |= there && !v;
                                if (!v) seen &= ~(1u << (((hv * 2 + r) * NT + nt) * 2 + e));
                            }
                    }
            }
            bool grew = false;
            float corr[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
            {
#pragma unroll
                for (int e = 0; e < 2; ++e)
                {
                    float x = -INFINITY;
#pragma unroll
                    for (int hv = 0; hv < HV; ++hv)
#pragma unroll
                        for (int r = 0; r < 2; ++r)
                        {
                            float& y = sc[hv][nt][2 * r + e];
                            y *= F16 ? fac[nt][e] * kf[hv][r] : fac[nt][e];
                            if (!whole && !((seen >> (((hv * 2 + r) * NT + nt) * 2 + e)) & 1u)) y = -INFINITY;
                            x = fmaxf(x, F16 ? y + ev[hv][r] : y);
                        }
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    corr[nt][e] = 1.f;
                    if (x > m[nt][e])
                    {
                        corr[nt][e] = exp2f(m[nt][e] - x);
                        m[nt][e] = x;
                        grew = true;
                    }
                    const float mm = m[nt][e] == -INFINITY ? 0.f : m[nt][e];
                    float sum = 0.f;
#pragma unroll
                    for (int hv = 0; hv < HV; ++hv)
#pragma unroll
                        for (int r = 0; r < 2; ++r)
                        {
                            float& y = sc[hv][nt][2 * r + e];
                            y = exp2f(y - mm);   // (a NaN score stays one)
                            sum += y;
                            // A scale of NaN must not meet a weight of zero that stands for "not seen".
                            if constexpr (F16)
                                y = (!whole && !((seen >> (((hv * 2 + r) * NT + nt) * 2 + e)) & 1u)) ? 0.f : y * vs[hv][r];
                        }
                    l[nt][e] = l[nt][e] * corr[nt][e] + sum;
                }
            }
            if (__any_sync(0xffffffffu, grew))
            {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < MTS; ++x)
                    {
                        acc[nt][x][0] *= corr[nt][0];
                        acc[nt][x][1] *= corr[nt][1];
                        acc[nt][x][2] *= corr[nt][0];
                        acc[nt][x][3] *= corr[nt][1];
                    }
            }
            // Values that some column must not see may be infinite or NaN, and 0 times those is NaN:
            // if there are any in such a step, its products are taken one by one.
            if constexpr (!F16)
            {
                if (__any_sync(0xffffffffu, hidden))
                {
                    bool odd = false;
                    for (int x = lane; x < KEYS * CPR; x += 32)
                    {
                        const uint4 w = lds128(vb + x * 16);
                        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            odd |= (ws[e] & 0x7f800000u) == 0x7f800000u || (sizeof(CT) == 2 && (ws[e] & 0x7f80u) == 0x7f80u);
                    }
                    if (__any_sync(0xffffffffu, odd))
                    {
#pragma unroll
                        for (int hr = 0; hr < 2 * HV; ++hr)
                        {
                            const unsigned char* const vst = ring + slot * Sh::STAGE + KEYS * RB;
#pragma unroll 1
                            for (int k = 0; k < 8; ++k)
                            {
                                const int row = 8 * hr + k, key = key_of(u0 + row);
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                    for (int e = 0; e < 2; ++e)
                                    {
                                        const float p = __shfl_sync(0xffffffffu, sc[hr >> 1][nt][2 * (hr & 1) + e], k * 4 + t);
                                        if (!((live >> row) & 1u) || !paged_sees(a, pos[nt][e], key)) continue;
#pragma unroll
                                        for (int x = 0; x < MTS; ++x)
#pragma unroll
                                            for (int hf = 0; hf < 2; ++hf)
                                            {
                                                const int by = split_dim<CT, D>(x, hf, g) * static_cast<int>(sizeof(CT));
                                                acc[nt][x][2 * hf + e] +=
                                                    p * to_f32<CT>(*reinterpret_cast<const CT*>(vst + split_v_at<CT, D>(row, by >> 4) + (by & 15)));
                                            }
                                    }
                            }
                        }
                        continue;
                    }
                }
            }
#pragma unroll
            for (int hv = 0; hv < HV; ++hv)
            {
                uint32_t pb[NT][2][NQ];   // weights as B fragments
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                {
                    uint32_t p0[NQ], p1[NQ];
                    split_pair<F16, NQ>(sc[hv][nt][0], sc[hv][nt][1], p0);
                    split_pair<F16, NQ>(sc[hv][nt][2], sc[hv][nt][3], p1);
#pragma unroll
                    for (int j = 0; j < NQ; ++j)
                    {
                        pb[nt][0][j] = movmatrix(p0[j]);
                        pb[nt][1][j] = movmatrix(p1[j]);
                    }
                }
                auto pv = [&](int mt, const uint32_t (&va)[NK][4]) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = NQ - 1; j >= 0; --j)
#pragma unroll
                            for (int n = NK - 1; n >= 0; --n)
                                if (n + j <= 2) mma16816<F16>(acc[nt][mt], va[n], pb[nt][0][j], pb[nt][1][j]);
                };
                if constexpr (sizeof(CT) == 2)
                {
#pragma unroll
                    for (int mt = 0; mt < MTS; ++mt)
                    {
                        uint32_t va[1][4];
                        ldmatrix4_trans(va[0], vb + split_v_at<CT, D>(16 * hv + (lane & 7) + ((lane >> 4) << 3), 2 * mt + ((lane >> 3) & 1)));
                        pv(mt, va);
                    }
                }
                else if constexpr (sizeof(CT) == 4)
                {
#pragma unroll
                    for (int x = 0; x < D / 32; ++x)
                    {
                        const int r0 = 16 * hv + 2 * t, c = 8 * x + g;
                        const uint4 f0 = lds128(vb + split_v_at<CT, D>(r0, c)), f1 = lds128(vb + split_v_at<CT, D>(r0 + 1, c));
                        const uint4 f2 = lds128(vb + split_v_at<CT, D>(r0 + 8, c)), f3 = lds128(vb + split_v_at<CT, D>(r0 + 9, c));
#pragma unroll
                        for (int y = 0; y < 2; ++y)
                        {
                            uint32_t va[NK][4], p[NK];
                            auto put = [&](int at, uint32_t lo, uint32_t hi) {
                                split_pair<false, NK>(__uint_as_float(lo), __uint_as_float(hi), p);
#pragma unroll
                                for (int n = 0; n < NK; ++n) va[n][at] = p[n];
                            };
                            put(0, y ? f0.z : f0.x, y ? f1.z : f1.x);
                            put(1, y ? f0.w : f0.y, y ? f1.w : f1.y);
                            put(2, y ? f2.z : f2.x, y ? f3.z : f3.x);
                            put(3, y ? f2.w : f2.y, y ? f3.w : f3.y);
                            pv(2 * x + y, va);
                        }
                    }
                }
                else
                {
                    // Rows 2t, 2t + 1, 2t + 8, 2t + 9; D / 8 consecutive dimensions of each.
                    constexpr int W = D / 32;   // words
                    uint32_t f[4][W];
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                    {
                        const int row = 16 * hv + 2 * t + (r & 1) + (r >> 1) * 8;
                        if constexpr (D == 128)
                        {
                            const uint4 x = lds128(vb + split_v_at<CT, D>(row, g));
                            f[r][0] = x.x; f[r][1] = x.y; f[r][2] = x.z; f[r][3] = x.w;
                        }
                        else
                        {
                            const uint2 x = lds64(vb + split_v_at<CT, D>(row, g >> 1) + (g & 1) * 8);
                            f[r][0] = x.x; f[r][1] = x.y;
                        }
                    }
#pragma unroll
                    for (int mt = 0; mt < MTS; ++mt)
                    {
                        const int wd = mt >> 1;
                        const uint32_t s0 = (mt & 1) ? 0x62u : 0x40u, s1 = (mt & 1) ? 0x73u : 0x51u;
                        uint32_t va[1][4];
                        va[0][0] = codes_f16<CT>(__byte_perm(f[0][wd], f[1][wd], s0));
                        va[0][1] = codes_f16<CT>(__byte_perm(f[0][wd], f[1][wd], s1));
                        va[0][2] = codes_f16<CT>(__byte_perm(f[2][wd], f[3][wd], s0));
                        va[0][3] = codes_f16<CT>(__byte_perm(f[2][wd], f[3][wd], s1));
                        pv(mt, va);
                    }
                }
            }
        }
        cp_wait<0>();

        // ---- the warps' parts into one ----
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
            {
                l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 4);
                l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 8);
                l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 16);
            }
        __syncthreads();   // every ring is drained
        float* const sums = reinterpret_cast<float*>(smem);                       // [warp][COLS][D + 4]
        float2* const ml = reinterpret_cast<float2*>(smem + Sh::ML_OFF);           // [warp][COLS]
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
            {
                const int c = nt * 8 + 2 * t + e;
                if (g == 0) ml[warp * COLS + c] = make_float2(m[nt][e], l[nt][e]);
                if (c < cols)
#pragma unroll
                    for (int x = 0; x < MTS; ++x)
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf)
                            sums[(warp * COLS + c) * (D + 4) + split_dim<CT, D>(x, hf, g)] = acc[nt][x][2 * hf + e];
            }
        __syncthreads();
        const bool complete = tile0 == 0 && tile1 == it.tiles;
        const int part_slot = 2 * blockIdx.x + (first ? 0 : 1);
        float* const part = parts + static_cast<long long>(part_slot) * Sh::PART;
        for (int x = tid; x < cols * (D / 4); x += kSplitThreads)
        {
            const int c = x / (D / 4), d = (x % (D / 4)) * 4;
            float2 w[kSplitWarps];
            float M = -INFINITY, L = 0.f, o[4] = {};
#pragma unroll
            for (int k = 0; k < kSplitWarps; ++k)
            {
                w[k] = ml[k * COLS + c];
                M = fmaxf(M, w[k].x);
            }
#pragma unroll
            for (int k = 0; k < kSplitWarps; ++k)
            {
                const float f = w[k].x == M ? 1.f : exp2f(w[k].x - M);
                const float4 v = *reinterpret_cast<const float4*>(sums + (k * COLS + c) * (D + 4) + d);
                L += f * w[k].y;
                o[0] += f * v.x; o[1] += f * v.y; o[2] += f * v.z; o[3] += f * v.w;
            }
            if (complete)
            {
                const float inv = L == 0.f ? 0.f : (F16 ? 1.f / 16384.f : 1.f) / L;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] *= inv;
                const int cc = it.tile * COLS + c, row = it.q.row0 + cc / a.group, h = it.head * a.group + cc % a.group;
                store_row<QT, 4>(a.out, row * a.o_row_stride + h * a.o_head_stride + d, o);
            }
            else
            {
                if (d == 0) reinterpret_cast<float2*>(part)[c] = make_float2(M, L);
                *reinterpret_cast<float4*>(part + 2 * COLS + c * D + d) = make_float4(o[0], o[1], o[2], o[3]);
            }
        }
        left -= n_tiles;
        if (!complete && tile0 == 0 && tid == 0)
        {
            // This CTA starts the item: its parts are here and in the CTAs up to the one with the item's last tile.
            const long long x_last = st.x1 - left - n_tiles + it.tiles - 1 - tile0;   // (global index of that tile)
            const int last = static_cast<int>(x_last / st.share);
            PagedJoin d;
            d.count = last - static_cast<int>(blockIdx.x) + 1;
            d.first_slot = part_slot;
            d.first_cta = blockIdx.x;
            d.row0 = it.q.row0;
            d.col0 = it.tile * COLS;
            d.cols = cols;
            d.head = it.head;
            d.pad = 0;
            *desc = d;
        }
        if (left == 0) break;
        first = false;
        // The next item: next head, next tile of columns, next sequence.
        tile0 = 0;
        if (++it.head == a.c.kv_heads)
        {
            it.head = 0;
            if (++it.tile >= split_row_tiles<COLS>(a, it.q.n))
            {
                it.tile = 0;
                do
                {
                    ++it.seq;
                } while (it.seq < a.b.num_seqs && (!paged_seq(a.b, it.seq, a.c.page_size, nullptr, it.q) || it.q.n == 0));
                if (it.seq >= a.b.num_seqs) break;   // (the arrays changed under the call)
            }
            it.w = paged_span(a, it.q, it.tile * COLS, COLS);
            it.tiles = split_tiles<Sh::TILE>(it.w.n);
        }
        __syncthreads();   // the sums were read; the ring is free
    }
}

// Joins the parts of the item that CTA blockIdx.x of the split kernel started, if it did.
template <typename QT, bool F16, int D, int NT>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedAttnArgs a)
{
    constexpr int COLS = 8 * NT, PART = COLS * (D + 2);
    pdl_wait();
    const PagedJoin j = static_cast<const PagedJoin*>(a.work)[blockIdx.x];
    if (j.count == 0) return;
    const float* const parts = reinterpret_cast<const float*>(static_cast<const unsigned char*>(a.work) + kSplitDescBytes);
    for (int x = threadIdx.x; x < j.cols * (D / 4); x += 128)
    {
        const int c = x / (D / 4), d = (x % (D / 4)) * 4;
        float M = -INFINITY, L = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        auto at = [&](int k) {
            return parts + static_cast<long long>(k == 0 ? j.first_slot : 2 * (j.first_cta + k)) * PART;
        };
        constexpr int U = 8;   // parts in flight
        for (int k0 = 0; k0 < j.count; k0 += U)
        {
            float2 w[U];
            float4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
            {
                const int k = min(k0 + u, j.count - 1);
                w[u] = reinterpret_cast<const float2*>(at(k))[c];
                v[u] = *reinterpret_cast<const float4*>(at(k) + 2 * COLS + c * D + d);
            }
            float top = M;
#pragma unroll
            for (int u = 0; u < U; ++u) top = fmaxf(top, w[u].x);
            const float f0 = M == top ? 1.f : exp2f(M - top);
            L *= f0;
            o.x *= f0; o.y *= f0; o.z *= f0; o.w *= f0;
#pragma unroll
            for (int u = 0; u < U; ++u)
            {
                if (k0 + u >= j.count) break;
                const float f = w[u].x == top ? 1.f : exp2f(w[u].x - top);
                L += f * w[u].y;
                o.x += f * v[u].x; o.y += f * v[u].y; o.z += f * v[u].z; o.w += f * v[u].w;
            }
            M = top;
        }
        const float inv = L == 0.f ? 0.f : (F16 ? 1.f / 16384.f : 1.f) / L;
        const float r[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
        const int cc = j.col0 + c, row = j.row0 + cc / a.group, h = j.head * a.group + cc % a.group;
        store_row<QT, 4>(a.out, row * a.o_row_stride + h * a.o_head_stride + d, r);
    }
}

}  // namespace hy
