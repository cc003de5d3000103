// Attention of a batch's rows over the paged cache.
//
// out = softmax(scale * q k^T) v over the positions that a row sees, in one
// pass over the keys: a running maximum m, the sum l of 2^(s - m) and the sum
// of 2^(s - m) v are kept in fp32 and rescaled when m grows (s in units of
// log 2). Parts of the keys are joined by the same rescaling.
//
// What a tile of rows sees is one run of "virtual" positions: the sinks before
// its window, then the window's positions up to the last row's; neither the
// gap between them nor what lies behind the last row is ever looked up. (The wide kernel of
// hy_paged_chunk.cuh fetches pages 16 rows at a time where they hold a multiple of 16.)
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
    int page_shift, group_shift;   // log2 of page_size and of group, or -1
    float scale_log2;     // scale * log2(e)
    void* work;           // workspace
};

// Row of column c.
__device__ __forceinline__ int paged_row_of(const PagedAttnArgs& a, int c) { return a.group_shift >= 0 ? c >> a.group_shift : c / a.group; }

// The keys that the columns [c0, c0 + cols) of a sequence see. A column is a
// (row, head of the group) pair: column c is row c / group.
struct PagedSpan {
    int p_first, p_last;   // positions of the first and last row
    int sinks, lo, n;      // virtual position u < sinks: u, else lo + u - sinks; n of them
};
// align (a power of two): the run's parts start and the sinks end at multiples of it (what that adds is masked).
// Above 1 only where it divides the page size: then what it adds lies in pages that hold visible keys too.
__device__ __forceinline__ PagedSpan paged_span(const PagedAttnArgs& a, const PagedSeq& s, int c0, int cols, int align = 1)
{
    PagedSpan o;
    const int last = min(s.n * a.group, c0 + cols) - 1;
    o.p_first = s.kv - s.n + paged_row_of(a, c0);
    o.p_last = s.kv - s.n + paged_row_of(a, last);
    const int hi = o.p_last < 0 ? 0 : a.causal ? o.p_last + 1 : s.kv;
    // (rows before position 0 see nothing: the first that may see something stands at 0 or later)
    o.lo = (a.window > 0) ? min(hi, max(0, max(0, o.p_first) - a.window + 1)) & -align : 0;
    o.sinks = a.sinks >= o.lo ? o.lo : (a.sinks + align - 1) & -align;
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

// 2^x, off by less than 2^-22; 0 below 2^-126.
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Exponent of a scale of values, of either sign, kept within 100 octaves.
__device__ __forceinline__ int scale_exponent(float v)
{
    return min(max(static_cast<int>((__float_as_uint(v) >> 23) & 0xffu) - 127, -100), 100);
}
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

// Two 8-bit codes of x, its low (HIGH: high) 16 bits, as a pair of f16 (exact for both types).
template <typename CT, bool HIGH = false>
__device__ __forceinline__ uint32_t codes_f16(uint32_t x)
{
    if constexpr (std::is_same_v<CT, E4M3>)
    {
        uint32_t y;
        if constexpr (HIGH) asm("{.reg .b16 t, u;\n\tmov.b32 {t, u}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, u;\n\t}" : "=r"(y) : "r"(x));
        else asm("{.reg .b16 t, u;\n\tmov.b32 {t, u}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(y) : "r"(x));
        return y;
    }
    else
    {
        // 0x6400 | (code ^ 0x80) is 1024 + 128 + code in f16.
        const uint32_t y = __byte_perm(x ^ 0x80808080u, 0x64646464u, HIGH ? 0x4342 : 0x4140);
        const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const __half2 z = __hsub2(*reinterpret_cast<const __half2*>(&y), bias);
        return *reinterpret_cast<const uint32_t*>(&z);
    }
}

// ---------------------------------------------------------------------------
// Few rows per sequence: the keys are split over the GPU.
//
// The work is the list of (sequence, tile of COLS columns, KV head) items, each
// of ceil(keys / TILE) tiles (at least one), T in all; CTA i of G takes the next
// ceil(T / G) tiles of the whole list, whatever items they belong to, so every CTA
// streams the same number of keys however ragged the lengths are. Memory bounds it
// (a key is used by the group's heads only), so all that matters is that loads
// never pause: every warp owns a quarter of a tile's keys and a cp.async ring of its
// own, and the warps meet only at the end of an item. 64 tokens over 1024-8192 E4M3
// keys each (613 MB): 109 us, 5.6 TB/s, in a run of a few calls, 117 us, 5.2 TB/s, back to back (the power
// limit holds the SM clock at 1.78 GHz); one token over 2048 fp32 keys: 11 us, of which the
// keys take 2.5 and the look-ups and joins around them the rest.
//
// A CTA's first and last items may be shared with its neighbours: those leave
// (m, l, sum) parts in the workspace, slot 2 i for the first item and 2 i + 1 for a
// later one, and paged_join_kernel adds up the parts of an item. The CTA that
// starts such an item leaves its description.
//
// What a step of a warp computes is an engine's: MmaEngine (tensor cores) or
// FmaEngine (fp32 caches and up to 4 columns).
// ---------------------------------------------------------------------------
constexpr int kSplitWarps = 4;
constexpr int kSplitThreads = kSplitWarps * 32;
constexpr int kSplitMaxCtas = 3 * 148;   // three CTAs per SM

struct PagedJoin {   // description of an item whose parts are joined; count 0: none
    int count, first_slot, first_cta, row0, col0, cols, head, pad;
};

// Bytes before the parts: the descriptions.
constexpr size_t kSplitDescBytes = kSplitMaxCtas * sizeof(PagedJoin);

struct SplitItem {
    PagedSeq q;
    PagedSpan w;
    int seq, tile, head, tiles;
    int cols;   // columns that are there
};
__device__ __forceinline__ int split_key(const SplitItem& it, int u) { return u < it.w.sinks ? u : it.w.lo + u - it.w.sinks; }
// Row tensor offset of column c of an item.
__device__ __forceinline__ long long split_q_at(const PagedAttnArgs& a, const SplitItem& it, int tile_cols, int c)
{
    const int cc = it.tile * tile_cols + c, row = paged_row_of(a, cc);
    return (it.q.row0 + row) * a.q_row_stride + (it.head * a.group + cc - row * a.group) * a.q_head_stride;
}
__device__ __forceinline__ int split_pos(const PagedAttnArgs& a, const SplitItem& it, int tile_cols, int c)
{
    return c < it.cols ? it.q.kv - it.q.n + paged_row_of(a, it.tile * tile_cols + c) : -1;
}
// Every column sees every one of the KEYS keys from u0 on (`live` tells which are there).
template <int KEYS>
__device__ __forceinline__ bool split_whole(const PagedAttnArgs& a, const SplitItem& it, int u0, uint32_t live)
{
    const int j_first = split_key(it, u0), j_last = split_key(it, min(u0 + KEYS - 1, it.w.n - 1));
    return live == (KEYS == 32 ? 0xffffffffu : (1u << (KEYS & 31)) - 1u) && it.w.p_first >= 0 &&
           (!a.causal || (j_last <= it.w.p_first &&
                          (a.window == 0 || j_first > it.w.p_last - a.window || j_last < a.sinks)));
}

// Sizes that follow from an engine's: ring stages and CTAs per SM. Three CTAs
// for narrow tiles (168 registers a thread), else two, else (16 KB a step) one.
template <typename E>
struct SplitShape {
    static constexpr int TILE = kSplitWarps * E::KEYS;
    static constexpr int STAGE = 2 * E::KEYS * E::RB;
    static constexpr int SCALES = E::F16 ? 2 * E::KEYS * 4 : 0;
    static constexpr int FIX = E::Q_SMEM + E::COLS * 4 + kSplitWarps * E::COLS * 8 + 256;
    static constexpr int fit(int kb, int most)
    {
        const int n = (kb * 1024 - FIX) / (kSplitWarps * (STAGE + SCALES + 4));
        return n < most ? n : most;
    }
    static constexpr int OCC = (E::MAX_OCC == 3 && fit(74, 4) >= 2) ? 3 : fit(112, 4) >= 2 ? 2 : 1;
    static constexpr int S = OCC == 3 ? fit(74, 4) : OCC == 2 ? fit(112, 4) : fit(224, 4);
    static constexpr int RING = kSplitWarps * S * STAGE;
    static constexpr int MERGE = kSplitWarps * E::COLS * (E::D + 4) * 4;   // the warps' sums, over the drained ring
    static constexpr int SC_OFF = RING > MERGE ? RING : MERGE;
    static constexpr int MASK_OFF = SC_OFF + kSplitWarps * S * SCALES;     // a bit for every key that is there
    static constexpr int Q_OFF = (MASK_OFF + kSplitWarps * S * 4 + 127) / 128 * 128;
    static constexpr int MAX_OFF = Q_OFF + E::Q_SMEM;                      // [COLS] bits of a column's largest |q|
    static constexpr int ML_OFF = (MAX_OFF + E::COLS * 4 + 7) / 8 * 8;     // [warps][COLS] (m, l)
    static constexpr int SMEM = ML_OFF + kSplitWarps * E::COLS * 8;
    static_assert(S >= 2 && SMEM <= 227 * 1024, "shared memory");
    static constexpr int GRID = 148 * OCC;
    static constexpr int PART = E::COLS * (E::D + 2);   // a part: [COLS] (m, l), then [COLS][D]
};

// ---------------------------------------------------------------------------
// The products on the tensor cores, taken transposed: S^T[key x column] = K Q^T
// and O^T[dim x column] = V^T P^T. With the columns in the 8-wide dimension a
// decode step of two heads wastes 6 of 8 lanes instead of 14 of 16, the
// accumulators of 128 dimensions are 32 registers, and a column's softmax state
// lies in the same lane for the scores and for the output.
//
// bf16 and fp32 caches multiply in bf16 (an fp32 number as three terms, products
// of terms i + j <= 2: the three left out are below 2^-21 together); 8-bit caches in f16, where their codes are
// exact and so is a bf16 query (each row times a power of two; what is below 2^-31 of its largest loses bits), fp32
// queries as two f16 terms. Which dimensions a lane takes from a row is free as long as q
// agrees, so 8-bit and fp32 keys are read from shared memory in 16-byte pieces.
//
// Decode steps are bound by memory; with 32 columns of fp32 queries the 192 products a
// warp's 16 keys take bound it (8 cycles each): 4 verify blocks of 16 rows at 2048 keys 27.3 us. Chunks of fp32
// rows, and of any rows over fp32 pages, stay here too, every 32 columns reading the keys anew: 4 x ~1012 rows over
// 6000-8192 keys take 2.2 ms (fp32 rows, BF16 pages), 1.9 (fp32, E4M3), 3.5 (bf16, F32) and 5.8 (fp32, F32).
// (Spills: 52 bytes a thread for fp32 rows over fp32 pages of 128 dimensions and 32 columns, 44 over BF16 pages, 48 to 100
// over 8-bit pages.)
// ---------------------------------------------------------------------------
template <typename QT_, typename CT_, int D_, int NT>
struct MmaEngine {
    using QT = QT_;
    using CT = CT_;
    static constexpr int D = D_, COLS = 8 * NT;
    static constexpr bool F16 = kCodes<CT>;
    static constexpr int NQ = std::is_same_v<QT, float> ? (F16 ? 2 : 3) : 1;   // terms of q and of the weights
    static constexpr int NK = std::is_same_v<CT, float> ? 3 : 1;               // terms of k and v
    static constexpr int RB = D * static_cast<int>(sizeof(CT));                // bytes of a row
    // Keys of a warp's step: 32 where that is 8 KB or less (the work that a step
    // costs whatever its keys - addresses, maxima, shuffles - is halved) and the registers allow it, else 16.
    static constexpr int KEYS = RB <= 128 && NT < 4 ? 32 : 16;
    static constexpr int MAX_OCC = NT == 1 ? 3 : 2;   // CTAs per SM that the registers allow
    static constexpr int KS = D / 16, MTS = D / 16, HV = KEYS / 16;
    static constexpr int Q_SMEM = KS * NT * NQ * 256;
    static constexpr int QI = KS * NT / kSplitWarps;                           // q fragments that a thread makes
    static constexpr bool QREG = KS * NT * 2 * NQ <= 32;                       // q stays in registers
    // Chains of products per score. The tensor cores cut a sum at every product, so the products of the second and third
    // terms, which hardly change it, have chains of their own (verify blocks over fp32 pages with loud dimensions: off by
    // 7.3e-7 instead of 4.1e-6, over BF16 pages 6.7e-7 instead of 2.0e-6; 27.1 -> 27.3 us).
    static constexpr int NA = NT >= 4 ? (NQ == 3 ? 2 : 1) : NQ * NK == 1 ? 2 : NQ > NK ? NQ : NK;
    static constexpr int MG = NT >= 4 ? 1 : 2;                                      // m tiles whose products alternate
    static constexpr float OUT = F16 ? 1.f / 16384.f : 1.f;                         // the sums' unit

    uint2 qreg[QREG ? NQ * KS * NT : 1];
    const uint2* qf;
    int pos[NT][2];       // positions and score factors of this lane's columns (2t, 2t + 1 of every n tile)
    float fac[NT][2];
    float m[NT][2], l[NT][2], acc[NT][MTS][4];

    // Where 16-byte piece c of key row r lies in a stage (bytes), for K and for V: the
    // rotations keep the lanes of each shared-memory phase on different banks.
    static __device__ __forceinline__ int k_at(int r, int c)
    {
        if constexpr (sizeof(CT) == 2) return r * RB + ((c ^ (r & 7)) << 4);
        else if constexpr (RB >= 128) return r * RB + ((c ^ ((r & 1) << 2)) << 4);
        else return r * RB + (c << 4);
    }
    static __device__ __forceinline__ int v_at(int r, int c)
    {
        if constexpr (sizeof(CT) == 2) return r * RB + ((c ^ (r & 7)) << 4);
        else if constexpr (RB >= 128) return r * RB + ((c ^ (r & 6)) << 4);
        else
        {
            // 64-byte rows: even rows first, so that rows 0, 2, 4, 6 span both halves of the banks.
            const int at = (r & ~7) | ((r & 1) << 2) | ((r & 6) >> 1);
            return at * RB + ((c ^ (at & 2)) << 4);
        }
    }
    // Output dimension of accumulator row (m tile, half) of lane group g, by how V's fragments are read.
    static __device__ __forceinline__ int dim_of(int mt, int half, int g)
    {
        if constexpr (sizeof(CT) == 4) return 32 * (mt >> 1) + 4 * g + 2 * (mt & 1) + half;
        else if constexpr (sizeof(CT) == 2) return 16 * mt + 8 * half + g;
        else return (D / 8) * g + 2 * mt + half;
    }

    // q of the fragments that this thread makes, straight from memory; fragment i of
    // thread tid: lane tid % 32 of n tile x % NT, k step x / NT, x = tid / 32 + 4 i.
    float raw[QI][4];
    __device__ __forceinline__ void fetch_q(const PagedAttnArgs& a, const SplitItem& it)
    {
        const int ln = threadIdx.x & 31, gg = ln >> 2, tt = ln & 3;
        long long at[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) at[nt] = split_q_at(a, it, COLS, min(nt * 8 + gg, it.cols - 1));
#pragma unroll
        for (int i = 0; i < QI; ++i)
        {
            const int x = (threadIdx.x >> 5) + kSplitWarps * i, nt = x % NT, ks = x / NT;
            const long long o = NT == 1 ? at[0] : at[nt % NT];
            if constexpr (sizeof(CT) == 2)
            {
                const QT* p = static_cast<const QT*>(a.q) + o + 16 * ks + 2 * tt;
                if constexpr (sizeof(QT) == 4)
                {
                    const float2 u = __ldg(reinterpret_cast<const float2*>(p)), w = __ldg(reinterpret_cast<const float2*>(p + 8));
                    raw[i][0] = u.x; raw[i][1] = u.y; raw[i][2] = w.x; raw[i][3] = w.y;
                }
                else
                {
                    const uint32_t u = __ldg(reinterpret_cast<const uint32_t*>(p)), w = __ldg(reinterpret_cast<const uint32_t*>(p + 8));
                    raw[i][0] = __uint_as_float(u << 16); raw[i][1] = __uint_as_float(u & 0xFFFF0000u);
                    raw[i][2] = __uint_as_float(w << 16); raw[i][3] = __uint_as_float(w & 0xFFFF0000u);
                }
            }
            else
            {
                load_row<QT, 4>(a.q, o + (sizeof(CT) == 4 ? 16 * ks + 4 * tt : 64 * (ks >> 2) + 16 * tt + 4 * (ks & 3)), raw[i]);
            }
            if (nt * 8 + gg >= it.cols) raw[i][0] = raw[i][1] = raw[i][2] = raw[i][3] = 0.f;
        }
    }
    // The fragments, through shared memory (all warps need all of them). colmax is zero on entry.
    __device__ __forceinline__ void make_q(const PagedAttnArgs& a, const SplitItem& it, unsigned char* smem_q, uint32_t* colmax)
    {
        const int ln = threadIdx.x & 31, gg = ln >> 2, t = ln & 3;
        uint2* const q = reinterpret_cast<uint2*>(smem_q);   // [term][ks][nt][lane]
        if constexpr (F16)
        {
            // A column's power of two: its largest magnitude comes to lie in [2^14, 2^15).
#pragma unroll
            for (int i = 0; i < QI; ++i)
            {
                uint32_t x = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) x = max(x, __float_as_uint(raw[i][e]) & 0x7fffffffu);
                x = max(x, __shfl_xor_sync(0xffffffffu, x, 1));
                x = max(x, __shfl_xor_sync(0xffffffffu, x, 2));
                if (t == 0) atomicMax(colmax + ((threadIdx.x >> 5) + kSplitWarps * i) % NT * 8 + gg, x);
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < QI; ++i)
        {
            const int x = (threadIdx.x >> 5) + kSplitWarps * i, nt = x % NT, ks = x / NT;
            if constexpr (F16)
            {
                const float up = __uint_as_float((254u << 23) - down_bits(colmax[nt * 8 + gg]));
#pragma unroll
                for (int e = 0; e < 4; ++e) raw[i][e] *= up;
            }
            uint32_t b0[NQ], b1[NQ];
            split_pair<F16, NQ>(raw[i][0], raw[i][1], b0);
            split_pair<F16, NQ>(raw[i][2], raw[i][3], b1);
#pragma unroll
            for (int j = 0; j < NQ; ++j) q[((j * KS + ks) * NT + nt) * 32 + ln] = make_uint2(b0[j], b1[j]);
        }
        __syncthreads();
        qf = q;
        if constexpr (QREG)
#pragma unroll
            for (int i = 0; i < NQ * KS * NT; ++i) qreg[i] = q[i * 32 + ln];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
        {
#pragma unroll
            for (int e = 0; e < 2; ++e)
            {
                const int c = nt * 8 + 2 * t + e;
                pos[nt][e] = split_pos(a, it, COLS, c);
                fac[nt][e] = F16 ? a.scale_log2 * __uint_as_float(down_bits(colmax[c])) : a.scale_log2;
                m[nt][e] = -INFINITY;
                l[nt][e] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < MTS; ++i) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
        }
    }
    // Bits of 2^-k, k = 14 - exponent of the largest magnitude, kept within the normal numbers.
    static __device__ __forceinline__ uint32_t down_bits(uint32_t largest)
    {
        return (min(max(largest >> 23, 16u), 254u) - 14u) << 23;
    }
    __device__ __forceinline__ uint2 q_frag(int term, int ks, int nt) const
    {
        const int i = (term * KS + ks) * NT + nt;
        if constexpr (QREG) return qreg[i];
        else return qf[i * 32 + (threadIdx.x & 31)];
    }

    // A step: KEYS keys of virtual positions u0 .., in shared memory at kb (keys, then values), scales at sc_u.
    __device__ __forceinline__ void step(const PagedAttnArgs& a, const SplitItem& it, int u0, uint32_t live,
                                         const unsigned char* stage, uint32_t kb, uint32_t sc_u)
    {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        const uint32_t vb = kb + KEYS * RB;
        // Scores of the step's keys: sc[hv][nt] holds keys 16 hv + g and + 8.
        float sc[HV][NT][4];
#pragma unroll
        for (int hv = 0; hv < HV; ++hv)
        {
            float part[NA][NT][4];   // chains of products that do not wait for one another
#pragma unroll
            for (int n = 0; n < NA; ++n)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) part[n][nt][0] = part[n][nt][1] = part[n][nt][2] = part[n][nt][3] = 0.f;
                uint4 w0, w1;   // 8-bit keys: 64 dimensions of rows g and g + 8
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
            {
                uint32_t ka[NK][4];
                if constexpr (sizeof(CT) == 2)
                {
                    ldmatrix4(ka[0], kb + k_at(16 * hv + (lane & 15), 2 * ks + (lane >> 4)));
                }
                else if constexpr (sizeof(CT) == 4)
                {
                    const uint4 x = lds128(kb + k_at(16 * hv + g, 4 * ks + t)),
                                y = lds128(kb + k_at(16 * hv + g + 8, 4 * ks + t));
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
                        w0 = lds128(kb + k_at(16 * hv + g, ks + t));
                        w1 = lds128(kb + k_at(16 * hv + g + 8, ks + t));
                    }
                    const uint32_t x = ks % 4 == 0 ? w0.x : ks % 4 == 1 ? w0.y : ks % 4 == 2 ? w0.z : w0.w;
                    const uint32_t y = ks % 4 == 0 ? w1.x : ks % 4 == 1 ? w1.y : ks % 4 == 2 ? w1.z : w1.w;
                    ka[0][0] = codes_f16<CT>(x);
                    ka[0][1] = codes_f16<CT>(y);
                    ka[0][2] = codes_f16<CT, true>(x);
                    ka[0][3] = codes_f16<CT, true>(y);
                }
#pragma unroll
                for (int j = NQ - 1; j >= 0; --j)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                    {
                        const uint2 b = q_frag(j, ks, nt);
#pragma unroll
                        for (int n = NK - 1; n >= 0; --n)
                            if (n + j <= 2)
                                mma16816<F16>(part[NQ * NK == 1 ? ks % NA : n + j < NA ? n + j : NA - 1][nt], ka[n], b.x, b.y);
                    }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                {
                    sc[hv][nt][e] = part[NA - 1][nt][e];   // the small terms first
#pragma unroll
                    for (int n = NA - 2; n >= 0; --n) sc[hv][nt][e] += part[n][nt][e];
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
                    const uint32_t at = sc_u + (16 * hv + 8 * r + g) * 4;
                    kf[hv][r] = lds_f32(at);
                    const float v = lds_f32(at + KEYS * 4);
                    // The maximum is taken over the score plus the exponent of the value's scale, so that
                    // a weight times its scale is below 2 and fits f16 (times 2^14).
                    ev[hv][r] = static_cast<float>(scale_exponent(v));
                    vs[hv][r] = v * 16384.f;
                }
            }
        const bool whole = split_whole<KEYS>(a, it, u0, live);
        uint32_t seen = 0xffffffffu;   // bit ((hv * 2 + r) * NT + nt) * 2 + e: the column sees the key
        bool hidden = false;           // some column does not see a key that was loaded
        if (!whole)
        {
#pragma unroll
            for (int hv = 0; hv < HV; ++hv)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                {
                    const int in16 = 16 * hv + 8 * r + g, j = split_key(it, u0 + in16);
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
                    corr[nt][e] = ex2(m[nt][e] - x);
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
                        y = ex2(y - mm);   // (a NaN score stays one)
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
                for (int x = lane; x < KEYS * RB / 16; x += 32)
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
                        const unsigned char* const vst = stage + KEYS * RB;
#pragma unroll 1
                        for (int k = 0; k < 8; ++k)
                        {
                            const int row = 8 * hr + k, key = split_key(it, u0 + row);
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
                                            const int by = dim_of(x, hf, g) * static_cast<int>(sizeof(CT));
                                            acc[nt][x][2 * hf + e] +=
                                                p * to_f32<CT>(*reinterpret_cast<const CT*>(vst + v_at(row, by >> 4) + (by & 15)));
                                        }
                                }
                        }
                    }
                    return;
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
            // The tensor cores cut sums, so that many of them one after another pull a sum toward zero: fp32 rows add up
            // a step's products by themselves and the steps by rounded additions (error where a warp adds up 250 steps:
            // 1.6e-5 -> 1.1e-6 over fp32 pages; verify blocks 26.0 -> 26.8 us, chunks over fp32 pages 5.2 -> 5.6 ms).
            auto pv = [&](int mt, const uint32_t (&va)[MG][NK][4]) {   // m tiles mt .. mt + MG - 1
                float sum[NQ > 1 ? MG : 1][NQ > 1 ? NT : 1][4];
                if constexpr (NQ > 1)
#pragma unroll
                    for (int x = 0; x < MG; ++x)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) sum[x][nt][0] = sum[x][nt][1] = sum[x][nt][2] = sum[x][nt][3] = 0.f;
#pragma unroll
                for (int j = NQ - 1; j >= 0; --j)
#pragma unroll
                    for (int n = NK - 1; n >= 0; --n)
#pragma unroll
                        for (int x = 0; x < MG; ++x)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                if (n + j <= 2)
                                {
                                    if constexpr (NQ > 1) mma16816<F16>(sum[x][nt], va[x][n], pb[nt][0][j], pb[nt][1][j]);
                                    else mma16816<F16>(acc[nt][mt + x], va[x][n], pb[nt][0][j], pb[nt][1][j]);
                                }
                if constexpr (NQ > 1)
#pragma unroll
                    for (int x = 0; x < MG; ++x)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[nt][mt + x][e] += sum[x][nt][e];
            };
            if constexpr (sizeof(CT) == 2)
            {
#pragma unroll
                for (int mt = 0; mt < MTS; mt += MG)
                {
                    uint32_t va[MG][1][4];
#pragma unroll
                    for (int x = 0; x < MG; ++x)
                        ldmatrix4_trans(va[x][0], vb + v_at(16 * hv + (lane & 7) + ((lane >> 4) << 3),
                                                                         2 * (mt + x) + ((lane >> 3) & 1)));
                    pv(mt, va);
                }
            }
            else if constexpr (sizeof(CT) == 4)
            {
#pragma unroll
                for (int x = 0; x < D / 32; ++x)
                {
                    const int r0 = 16 * hv + 2 * t, c = 8 * x + g;
                    const uint4 f0 = lds128(vb + v_at(r0, c)), f1 = lds128(vb + v_at(r0 + 1, c));
                    const uint4 f2 = lds128(vb + v_at(r0 + 8, c)), f3 = lds128(vb + v_at(r0 + 9, c));
#pragma unroll
                    for (int y0 = 0; y0 < 2; y0 += MG)
                    {
                        uint32_t va[MG][NK][4], p[NK];
#pragma unroll
                        for (int y = y0; y < y0 + MG; ++y)
                        {
                            auto put = [&](int at, uint32_t lo, uint32_t hi) {
                                split_pair<false, NK>(__uint_as_float(lo), __uint_as_float(hi), p);
#pragma unroll
                                for (int n = 0; n < NK; ++n) va[y - y0][n][at] = p[n];
                            };
                            put(0, y ? f0.z : f0.x, y ? f1.z : f1.x);
                            put(1, y ? f0.w : f0.y, y ? f1.w : f1.y);
                            put(2, y ? f2.z : f2.x, y ? f3.z : f3.x);
                            put(3, y ? f2.w : f2.y, y ? f3.w : f3.y);
                        }
                        pv(2 * x + y0, va);
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
                        const uint4 x = lds128(vb + v_at(row, g));
                        f[r][0] = x.x; f[r][1] = x.y; f[r][2] = x.z; f[r][3] = x.w;
                    }
                    else
                    {
                        const uint2 x = lds64(vb + v_at(row, g >> 1) + (g & 1) * 8);
                        f[r][0] = x.x; f[r][1] = x.y;
                    }
                }
#pragma unroll
                for (int mt = 0; mt < MTS; mt += MG)
                {
                    uint32_t va[MG][1][4];
#pragma unroll
                    for (int x = 0; x < MG; ++x)
                    {
                        const int wd = (mt + x) >> 1;
                        const uint32_t s0 = ((mt + x) & 1) ? 0x62u : 0x40u, s1 = ((mt + x) & 1) ? 0x73u : 0x51u;
                        va[x][0][0] = codes_f16<CT>(__byte_perm(f[0][wd], f[1][wd], s0));
                        va[x][0][1] = codes_f16<CT>(__byte_perm(f[0][wd], f[1][wd], s1));
                        va[x][0][2] = codes_f16<CT>(__byte_perm(f[2][wd], f[3][wd], s0));
                        va[x][0][3] = codes_f16<CT>(__byte_perm(f[2][wd], f[3][wd], s1));
                    }
                    pv(mt, va);
                }
            }
        }
    }

    // This warp's part: (m, l) of the columns, and their sums [COLS][D + 4].
    __device__ __forceinline__ void put(int cols, float* sums, float2* ml)
    {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
            {
                l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 4);
                l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 8);
                l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 16);
                const int c = nt * 8 + 2 * t + e;
                if (g == 0) ml[c] = make_float2(m[nt][e], l[nt][e]);
                if (c >= cols) continue;
#pragma unroll
                for (int x = 0; x < MTS; ++x)
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) sums[c * (D + 4) + dim_of(x, hf, g)] = acc[nt][x][2 * hf + e];
            }
    }
};

// ---------------------------------------------------------------------------
// fp32 caches, up to 4 columns: plain fp32 multiply-adds. Splitting an fp32 key
// into terms for the tensor cores costs a lane some 700 operations a step of 16 keys, the
// multiply-adds of two columns 256. Eight lanes share a key (each D / 8 of its dimensions in 16-byte
// pieces), the warp takes four keys at a time; each group of eight lanes keeps
// a softmax state of its own.
// ---------------------------------------------------------------------------
template <typename QT_, int D_, int NC>
struct FmaEngine {
    using QT = QT_;
    using CT = float;
    static constexpr int D = D_, COLS = NC;
    static constexpr bool F16 = false;
    static constexpr int RB = D * 4, KEYS = 4096 / RB, Q_SMEM = 0;   // a step is 8 KB
    static constexpr int MAX_OCC = D * NC > 256 ? 2 : 3;
    static constexpr int P = D / 32, KK = KEYS / 4;                   // 16-byte pieces of a lane; keys of a group
    static constexpr float OUT = 1.f;

    float4 q[NC][P], acc[NC][P];
    int pos[NC];
    float m[NC], l[NC];

    static __device__ __forceinline__ int k_at(int r, int c) { return r * RB + (c << 4); }
    static __device__ __forceinline__ int v_at(int r, int c) { return r * RB + (c << 4); }

    __device__ __forceinline__ void fetch_q(const PagedAttnArgs& a, const SplitItem& it)
    {
        const int dl = threadIdx.x & 7;
#pragma unroll
        for (int c = 0; c < NC; ++c)
        {
            const long long at = split_q_at(a, it, NC, min(c, it.cols - 1));
#pragma unroll
            for (int p = 0; p < P; ++p)
            {
                float x[4];
                load_row<QT, 4>(a.q, at + (dl + 8 * p) * 4, x);
                q[c][p] = make_float4(x[0], x[1], x[2], x[3]);
            }
        }
    }
    __device__ __forceinline__ void make_q(const PagedAttnArgs& a, const SplitItem& it, unsigned char*, uint32_t*)
    {
#pragma unroll
        for (int c = 0; c < NC; ++c)
        {
            pos[c] = split_pos(a, it, NC, c);
            m[c] = -INFINITY;
            l[c] = 0.f;
#pragma unroll
            for (int p = 0; p < P; ++p) acc[c][p] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }

    __device__ __forceinline__ void step(const PagedAttnArgs& a, const SplitItem& it, int u0, uint32_t live,
                                         const unsigned char*, uint32_t kb, uint32_t)
    {
        const int lane = threadIdx.x & 31, dl = lane & 7, kg = lane >> 3;
        float s[KK][NC];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
        {
#pragma unroll
            for (int c = 0; c < NC; ++c) s[kk][c] = 0.f;
#pragma unroll
            for (int p = 0; p < P; ++p)
            {
                const uint4 x = lds128(kb + k_at(4 * kk + kg, dl + 8 * p));
#pragma unroll
                for (int c = 0; c < NC; ++c)
                    s[kk][c] += dot4(q[c][p], make_float4(__uint_as_float(x.x), __uint_as_float(x.y), __uint_as_float(x.z), __uint_as_float(x.w)));
            }
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1)
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int c = 0; c < NC; ++c) s[kk][c] += __shfl_xor_sync(0xffffffffu, s[kk][c], o);
        const bool whole = split_whole<KEYS>(a, it, u0, live);
        uint32_t seen = 0xffffffffu;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int c = 0; c < NC; ++c)
            {
                s[kk][c] *= a.scale_log2;
                if (!whole && !(((live >> (4 * kk + kg)) & 1u) && paged_sees(a, pos[c], split_key(it, u0 + 4 * kk + kg))))
                {
                    s[kk][c] = -INFINITY;
                    seen &= ~(1u << (kk * NC + c));
                }
            }
#pragma unroll
        for (int c = 0; c < NC; ++c)
        {
            float top = s[0][c];
#pragma unroll
            for (int kk = 1; kk < KK; ++kk) top = fmaxf(top, s[kk][c]);
            float corr = 1.f;
            if (top > m[c])
            {
                corr = ex2(m[c] - top);
                m[c] = top;
#pragma unroll
                for (int p = 0; p < P; ++p)
                {
                    acc[c][p].x *= corr; acc[c][p].y *= corr; acc[c][p].z *= corr; acc[c][p].w *= corr;
                }
            }
            const float mm = m[c] == -INFINITY ? 0.f : m[c];
            l[c] *= corr;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
            {
                s[kk][c] = ex2(s[kk][c] - mm);   // (a NaN score stays one)
                l[c] += s[kk][c];
            }
        }
        const uint32_t vb = kb + KEYS * RB;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int p = 0; p < P; ++p)
            {
                const uint4 x = lds128(vb + v_at(4 * kk + kg, dl + 8 * p));
#pragma unroll
                for (int c = 0; c < NC; ++c)
                {
                    // (what a column does not see may hold anything: it is not even multiplied by 0)
                    if (!whole && !((seen >> (kk * NC + c)) & 1u)) continue;
                    acc[c][p].x = fmaf(s[kk][c], __uint_as_float(x.x), acc[c][p].x);
                    acc[c][p].y = fmaf(s[kk][c], __uint_as_float(x.y), acc[c][p].y);
                    acc[c][p].z = fmaf(s[kk][c], __uint_as_float(x.z), acc[c][p].z);
                    acc[c][p].w = fmaf(s[kk][c], __uint_as_float(x.w), acc[c][p].w);
                }
            }
    }

    __device__ __forceinline__ void put(int cols, float* sums, float2* ml)
    {
        const int lane = threadIdx.x & 31, dl = lane & 7;
#pragma unroll
        for (int c = 0; c < NC; ++c)
        {
            float top = m[c];
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const float f = m[c] == top ? 1.f : ex2(m[c] - top);
            auto all = [&](float x) {
                x *= f;
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                return x + __shfl_xor_sync(0xffffffffu, x, 16);
            };
            l[c] = all(l[c]);
            if (lane == 0) ml[c] = make_float2(top, l[c]);
#pragma unroll
            for (int p = 0; p < P; ++p)
            {
                const float4 v = make_float4(all(acc[c][p].x), all(acc[c][p].y), all(acc[c][p].z), all(acc[c][p].w));
                if (lane < 8 && c < cols) *reinterpret_cast<float4*>(sums + c * (D + 4) + (dl + 8 * p) * 4) = v;
            }
        }
    }
};

// ---------------------------------------------------------------------------
// The schedule.
// ---------------------------------------------------------------------------
template <int COLS>
__device__ __forceinline__ int split_row_tiles(const PagedAttnArgs& a, int n)
{
    return (n * a.group + COLS - 1) / COLS;
}
template <int TILE>
__device__ __forceinline__ int split_tiles(int keys) { return max(1, (keys + TILE - 1) / TILE); }

// x / n where the quotient is small; 32-bit arithmetic where it reaches.
__device__ __forceinline__ int split_div(long long x, int n)
{
    return x >> 31 ? static_cast<int>(x / n) : static_cast<int>(x) / n;
}

// Tiles of sequence s, all its items.
template <int COLS, int TILE>
__device__ __forceinline__ long long split_cost(const PagedAttnArgs& a, int s, int align)
{
    PagedSeq q;
    if (s >= a.b.num_seqs || !paged_seq(a.b, s, a.c.page_size, a.c.status, q)) return 0;
    long long c = 0;
    const int rt = split_row_tiles<COLS>(a, q.n);
    for (int t = 0; t < rt; ++t) c += split_tiles<TILE>(paged_span(a, q, t * COLS, COLS, align).n);
    return c * a.c.kv_heads;
}

// What the CTA takes of the list, and the sequence it starts in; every thread returns the same.
// Where a few sequences of one tile of columns each make fewer items than CTAs, the list is counted in units of
// several tiles of one item, so many that there are no more units than CTAs: every CTA has one unit, and none
// begins a second item, whose loads would start from nothing (some 5 us). Otherwise the unit is a tile and a CTA
// takes the next share of them.
struct SplitStart {
    long long x0, x1, total;   // the CTA's units; of all
    long long in_seq;          // x0 counted from its sequence's first unit
    long long share;           // units per CTA (1 where unit > 1)
    int unit;                  // tiles per unit
    int seq;
};
// By every warp for itself; true if the list is of that kind.
template <int COLS, int TILE>
__device__ __forceinline__ bool split_start_few(const PagedAttnArgs& a, int align, SplitStart& o)
{
    const int lane = threadIdx.x & 31, ctas = gridDim.x, h = a.c.kv_heads;
    PagedSeq q = {0, 0, 0};
    const bool there = lane < a.b.num_seqs && paged_seq(a.b, lane, a.c.page_size, a.c.status, q) && q.n > 0;
    const int t = there ? split_tiles<TILE>(paged_span(a, q, 0, COLS, align).n) : 0;
    const int all = __reduce_add_sync(0xffffffffu, min(t, 1 << 20));
    const int items = __popc(__ballot_sync(0xffffffffu, there)) * h;
    if (__any_sync(0xffffffffu, there && (q.n > COLS || q.n * a.group > COLS)) || items > ctas || all > (1 << 20) / h) return false;
    int unit = max(1, (all * h + ctas - 1) / ctas), mine = 0, total = 0;
    for (int tries = 0;; ++tries, ++unit)
    {
        if (tries == 6) return false;
        mine = (t + unit - 1) / unit * h;
        total = __reduce_add_sync(0xffffffffu, mine);
        if (total <= ctas) break;
    }
    int inc = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1)
    {
        const int v = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += v;
    }
    const int x = blockIdx.x;
    const unsigned in = __ballot_sync(0xffffffffu, x >= inc - mine && x < inc);
    o.total = total;
    o.share = 1;
    o.unit = unit;
    o.x0 = min(x, total);
    o.x1 = min(x + 1, total);
    o.seq = max(__ffs(in) - 1, 0);
    o.in_seq = x - __shfl_sync(0xffffffffu, inc - mine, o.seq);
    return true;
}
// scan: shared memory for a long long per warp and one more.
template <int COLS, int TILE, int THREADS>
__device__ __forceinline__ SplitStart split_start(const PagedAttnArgs& a, long long* scan, int align = 1)
{
    constexpr int WARPS = THREADS / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __shared__ int s_seq;
    SplitStart o;
    if (a.b.num_seqs <= 32 && split_start_few<COLS, TILE>(a, align, o)) return o;
    o.unit = 1;
    o.total = 0;
    const int rounds = (a.b.num_seqs + THREADS - 1) / THREADS;
    long long mine = 0;
    for (int r = 0; r < rounds; ++r)
    {
        mine = split_cost<COLS, TILE>(a, r * THREADS + tid, align);
        o.total += mine;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) o.total += __shfl_xor_sync(0xffffffffu, o.total, d);
    if (lane == 0) scan[warp] = o.total;
    __syncthreads();
    o.total = 0;
    for (int w = 0; w < WARPS; ++w) o.total += scan[w];
    o.share = max(1ll, (o.total + gridDim.x - 1) / gridDim.x);
    o.x0 = min(o.total, o.share * blockIdx.x);
    o.x1 = min(o.total, o.x0 + o.share);
    o.seq = 0;
    o.in_seq = 0;
    if (o.x0 >= o.x1) return o;
    long long base = 0;
    for (int r = 0; r < rounds; ++r)
    {
        if (rounds > 1) mine = split_cost<COLS, TILE>(a, r * THREADS + tid, align);
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
        for (int w = 0; w < WARPS; ++w) base += scan[w];
        const long long lo = before + inc - mine;
        if (o.x0 >= lo && o.x0 < lo + mine)
        {
            s_seq = r * THREADS + tid;
            scan[WARPS] = o.x0 - lo;
        }
        if (o.x0 < base) break;   // uniform: found in this round
    }
    __syncthreads();
    o.seq = s_seq;
    o.in_seq = scan[WARPS];
    return o;
}

template <typename E>
__global__ void __launch_bounds__(kSplitThreads, SplitShape<E>::OCC) paged_split_kernel(const PagedAttnArgs a)
{
    using Sh = SplitShape<E>;
    using CT = typename E::CT;
    using QT = typename E::QT;
    constexpr int COLS = E::COLS, S = Sh::S, RB = E::RB, CPR = RB / 16, KEYS = E::KEYS, TILE = Sh::TILE, D = E::D;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ long long scan[kSplitWarps + 1];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    PagedJoin* const desc = static_cast<PagedJoin*>(a.work) + blockIdx.x;
    float* const parts = reinterpret_cast<float*>(static_cast<unsigned char*>(a.work) + kSplitDescBytes);
    uint32_t* const colmax = reinterpret_cast<uint32_t*>(smem + Sh::MAX_OFF);
    if (tid < COLS) colmax[tid] = 0;
    if constexpr (E::F16) __syncthreads();   // before any warp's maxima (split_start may hold no barrier)
    pdl_wait();
    pdl_launch();

    const SplitStart st = split_start<COLS, TILE, kSplitThreads>(a, scan);
    if (tid == 0) desc->count = 0;   // (rewritten below, by the same thread, if an item's parts are to be joined)
    if (st.x0 >= st.x1) return;

    // The first item.
    SplitItem it;
    it.seq = st.seq;
    if (!paged_seq(a.b, it.seq, a.c.page_size, nullptr, it.q)) return;   // (the arrays changed under the call)
    long long in = st.in_seq;
    int units;
    for (it.tile = 0;; ++it.tile)
    {
        it.w = paged_span(a, it.q, it.tile * COLS, COLS);
        it.tiles = split_tiles<TILE>(it.w.n);
        units = (it.tiles + st.unit - 1) / st.unit;
        if (in < static_cast<long long>(units) * a.c.kv_heads) break;
        if ((it.tile + 1) * COLS >= it.q.n * a.group) return;   // (the arrays changed under the call)
        in -= static_cast<long long>(units) * a.c.kv_heads;
    }
    it.head = split_div(in, units);
    int tile0 = static_cast<int>(in - static_cast<long long>(it.head) * units) * st.unit;

    unsigned char* const ring = smem + warp * S * Sh::STAGE;
    const uint32_t ring_u = smem_u32(ring);
    const uint32_t sc_u = smem_u32(smem + Sh::SC_OFF + warp * S * Sh::SCALES);
    volatile uint32_t* const masks = reinterpret_cast<volatile uint32_t*>(smem + Sh::MASK_OFF) + warp * S;

    long long left = (st.x1 - st.x0) * st.unit;   // tiles
    bool first = true;
    E eng;
    while (true)
    {
        const int tile1 = static_cast<int>(min(static_cast<long long>(it.tiles), tile0 + left));
        const int n_tiles = tile1 - tile0;
        it.cols = min(COLS, it.q.n * a.group - it.tile * COLS);
        const int* const table = a.b.table + it.seq * a.b.table_stride;

        // ---- loads: this warp's keys of tile tile0 + i into slot i % S ----
        const int kr = lane % KEYS;
        // Page and row in it of this lane's key of a tile: looked up ahead of the load.
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
                const int slot = i % S;
                const bool live = (tile0 + i) * TILE + warp * KEYS + kr < it.w.n;
                const bool ok = live && pg >= 0 && pg < a.c.num_pages;
                if (live && !ok) paged_status(a.c.status, kPagedBadPage);
                const long long off = ok ? pg * a.c.page_stride + row * a.c.row_stride + it.head * a.c.head_stride : 0;
                uint32_t mask = __ballot_sync(0xffffffffu, ok);
                if constexpr (KEYS < 32) mask &= (1u << KEYS) - 1u;
                if (lane == 0) masks[slot] = mask;
                const uint32_t base = ring_u + slot * Sh::STAGE;
#pragma unroll
                for (int x = 0; x < KEYS * CPR / 32; ++x)
                {
                    const int idx = x * 32 + lane, r = idx / CPR, c = idx % CPR;
                    const long long o = __shfl_sync(0xffffffffu, off, r) + c * (16 / static_cast<int>(sizeof(CT)));
                    const bool pr = (mask >> r) & 1u;
                    cp_async16_zfill(base + E::k_at(r, c), static_cast<const CT*>(a.c.k) + o, pr);
                    cp_async16_zfill(base + KEYS * RB + E::v_at(r, c), static_cast<const CT*>(a.c.v) + o, pr);
                }
                if constexpr (E::F16)
                {
                    const long long so = ok ? pg * a.c.s_page_stride + row * a.c.s_row_stride + it.head * a.c.s_head_stride : 0;
                    const uint32_t dst = sc_u + slot * Sh::SCALES + kr * 4;
                    cp_async4_zfill(dst, a.c.k_scale + so, ok);
                    cp_async4_zfill(dst + KEYS * 4, a.c.v_scale + so, ok);
                }
            }
            cp_commit();
        };
        int pg[S] = {}, row[S] = {};
#pragma unroll
        for (int i = 0; i < S; ++i) look_up(i, pg[i], row[i]);
        eng.fetch_q(a, it);
#pragma unroll
        for (int i = 0; i < S - 1; ++i) load(i, pg[i], row[i]);
        int pg_next = pg[S - 1], row_next = row[S - 1];
        eng.make_q(a, it, smem + Sh::Q_OFF, colmax);

        // ---- the keys ----
        for (int i = 0; i < n_tiles; ++i)
        {
            cp_wait<S - 2>();
            __syncwarp();
            load(i + S - 1, pg_next, row_next);
            look_up(i + S, pg_next, row_next);
            const int u0 = (tile0 + i) * TILE + warp * KEYS;
            if (u0 >= it.w.n) continue;   // nothing for this warp in the item's last tile
            const int slot = i % S;
            eng.step(a, it, u0, masks[slot], ring + slot * Sh::STAGE, ring_u + slot * Sh::STAGE, sc_u + slot * Sh::SCALES);
        }
        cp_wait<0>();

        // ---- the warps' parts into one ----
        __syncthreads();   // every ring is drained
        float* const sums = reinterpret_cast<float*>(smem);                // [warp][COLS][D + 4]
        float2* const ml = reinterpret_cast<float2*>(smem + Sh::ML_OFF);   // [warp][COLS]
        eng.put(it.cols, sums + warp * COLS * (D + 4), ml + warp * COLS);
        __syncthreads();
        const bool complete = tile0 == 0 && tile1 == it.tiles;
        const int part_slot = 2 * blockIdx.x + (first ? 0 : 1);
        float* const part = parts + static_cast<long long>(part_slot) * Sh::PART;
        if (tid < COLS)
        {
            colmax[tid] = 0;
            // A column's joint (m, l), and the warps' factors in the place of their (m, l).
            float2 w[kSplitWarps];
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int k = 0; k < kSplitWarps; ++k)
            {
                w[k] = ml[k * COLS + tid];
                M = fmaxf(M, w[k].x);
            }
#pragma unroll
            for (int k = 0; k < kSplitWarps; ++k)
            {
                w[k].x = w[k].x == M ? 1.f : ex2(w[k].x - M);
                L += w[k].x * w[k].y;
            }
            const float inv = !complete ? 1.f : L == 0.f ? 0.f : E::OUT / L;
#pragma unroll
            for (int k = 0; k < kSplitWarps; ++k) ml[k * COLS + tid].x = w[k].x * inv;
            if (!complete && tid < it.cols) reinterpret_cast<float2*>(part)[tid] = make_float2(M, L);
        }
        __syncthreads();
#pragma unroll 2
        for (int x = tid; x < it.cols * (D / 4); x += kSplitThreads)
        {
            const int c = x / (D / 4), d = (x % (D / 4)) * 4;
            float o[4] = {};
#pragma unroll
            for (int k = 0; k < kSplitWarps; ++k)
            {
                const float f = ml[k * COLS + c].x;
                const float4 v = *reinterpret_cast<const float4*>(sums + (k * COLS + c) * (D + 4) + d);
                o[0] += f * v.x; o[1] += f * v.y; o[2] += f * v.z; o[3] += f * v.w;
            }
            if (complete)
            {
                const int cc = it.tile * COLS + c, rw = paged_row_of(a, cc);
                store_row<QT, 4>(a.out, (it.q.row0 + rw) * a.o_row_stride + (it.head * a.group + cc - rw * a.group) * a.o_head_stride + d, o);
            }
            else
            {
                *reinterpret_cast<float4*>(part + 2 * COLS + c * D + d) = make_float4(o[0], o[1], o[2], o[3]);
            }
        }
        left -= n_tiles;
        if (!complete && tile0 == 0 && tid == 0)
        {
            // This CTA starts the item: its parts are here and in the CTAs up to the one with the item's last tile.
            PagedJoin d;
            if (st.unit > 1) d.count = units;
            else d.count = static_cast<int>((st.x1 - left - n_tiles + it.tiles - 1) / st.share) - static_cast<int>(blockIdx.x) + 1;
            d.first_slot = part_slot;
            d.first_cta = blockIdx.x;
            d.row0 = it.q.row0;
            d.col0 = it.tile * COLS;
            d.cols = it.cols;
            d.head = it.head;
            d.pad = 0;
            *desc = d;
        }
        if (left == 0 || st.unit > 1) break;
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
            it.tiles = split_tiles<TILE>(it.w.n);
        }
        __syncthreads();   // the sums were read; the ring is free
    }
}

// Joins the parts of the item that CTA blockIdx.x of the split kernel started, if it
// did; blockIdx.y takes 8 of its columns. A float4 of a column is a group of D / 4 threads'; the
// groups are dealt to the columns that there are, several to a column where
// columns are few, each adding up every so manyth part.
constexpr int kJoinThreads = 512;
template <typename E>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const PagedAttnArgs a)
{
    constexpr int COLS = E::COLS, D = E::D, PART = COLS * (D + 2), LANES = D / 4, GROUPS = kJoinThreads / LANES;
    __shared__ float2 ml[GROUPS];
    __shared__ float4 vec[GROUPS][LANES];
    pdl_wait();
    const PagedJoin j = static_cast<const PagedJoin*>(a.work)[blockIdx.x];
    const int c0 = blockIdx.y * 8, cols = min(8, j.cols - c0);
    if (j.count == 0 || cols <= 0) return;
    const float* const parts = reinterpret_cast<const float*>(static_cast<const unsigned char*>(a.work) + kSplitDescBytes);
    const int grp = threadIdx.x / LANES, d = (threadIdx.x % LANES) * 4;
    const int width = cols <= 1 ? 1 : cols <= 2 ? 2 : cols <= 4 ? 4 : 8;   // columns, rounded up to a power of two
    const int per = GROUPS / width, c = c0 + grp % width, sub = grp / width;
    float M = -INFINITY, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto at = [&](int k) { return parts + static_cast<long long>(k == 0 ? j.first_slot : 2 * (j.first_cta + k)) * PART; };
    constexpr int U = 8;   // parts in flight
    if (c < c0 + cols)
    {
        for (int k0 = sub; k0 < j.count; k0 += U * per)
        {
            float2 w[U];
            float4 v[U];
#pragma unroll
            for (int x = 0; x < U; ++x)
            {
                if (k0 + x * per >= j.count) break;
                w[x] = reinterpret_cast<const float2*>(at(k0 + x * per))[c];
                v[x] = *reinterpret_cast<const float4*>(at(k0 + x * per) + 2 * COLS + c * D + d);
            }
            float top = M;
#pragma unroll
            for (int x = 0; x < U; ++x)
                if (k0 + x * per < j.count) top = fmaxf(top, w[x].x);
            const float f0 = M == top ? 1.f : ex2(M - top);
            L *= f0;
            o.x *= f0; o.y *= f0; o.z *= f0; o.w *= f0;
#pragma unroll
            for (int x = 0; x < U; ++x)
            {
                if (k0 + x * per >= j.count) break;
                const float f = w[x].x == top ? 1.f : ex2(w[x].x - top);
                L += f * w[x].y;
                o.x += f * v[x].x; o.y += f * v[x].y; o.z += f * v[x].z; o.w += f * v[x].w;
            }
            M = top;
        }
    }
    if (d == 0) ml[grp] = make_float2(M, L);
    vec[grp][d / 4] = o;
    __syncthreads();
    if (sub != 0 || c >= c0 + cols) return;
    float top = -INFINITY;
    for (int x = 0; x < per; ++x) top = fmaxf(top, ml[grp + x * width].x);
    L = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int x = 0; x < per; ++x)
    {
        const float2 w = ml[grp + x * width];
        const float f = w.x == top ? 1.f : ex2(w.x - top);
        const float4 v = vec[grp + x * width][d / 4];
        L += f * w.y;
        o.x += f * v.x; o.y += f * v.y; o.z += f * v.z; o.w += f * v.w;
    }
    const float inv = L == 0.f ? 0.f : E::OUT / L;
    const float r[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    const int cc = j.col0 + c, rw = paged_row_of(a, cc);
    store_row<typename E::QT, 4>(a.out, (j.row0 + rw) * a.o_row_stride + (j.head * a.group + cc - rw * a.group) * a.o_head_stride + d, r);
}

// The same for tiles of 256 columns, where many items are shared by two or three
// CTAs: blockIdx.y takes an eighth of the item's D / 4 x columns float4s, a thread two of them.
template <typename E>
__global__ void __launch_bounds__(kJoinThreads) paged_join_wide_kernel(const PagedAttnArgs a)
{
    constexpr int COLS = E::COLS, D = E::D, PART = COLS * (D + 2), LANES = D / 4, N = COLS * LANES / 8 / kJoinThreads;
    static_assert(N >= 1 && N * 8 * kJoinThreads == COLS * LANES, "shares");
    pdl_wait();
    const PagedJoin j = static_cast<const PagedJoin*>(a.work)[blockIdx.x];
    if (j.count == 0) return;
    const float* const parts = reinterpret_cast<const float*>(static_cast<const unsigned char*>(a.work) + kSplitDescBytes);
    float M[N], L[N];
    float4 o[N];
#pragma unroll
    for (int x = 0; x < N; ++x)
    {
        M[x] = -INFINITY;
        L[x] = 0.f;
        o[x] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const int e0 = blockIdx.y * (N * kJoinThreads) + threadIdx.x;   // element x: e0 + x * kJoinThreads
    if (e0 / LANES >= j.cols) return;
    constexpr int U = 4;   // parts in flight
    for (int k0 = 0; k0 < j.count; k0 += U)
    {
        float2 w[U][N];
        float4 v[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u)
        {
            const int k = min(k0 + u, j.count - 1);
            const float* const p = parts + static_cast<long long>(k == 0 ? j.first_slot : 2 * (j.first_cta + k)) * PART;
#pragma unroll
            for (int x = 0; x < N; ++x)
            {
                const int e = e0 + x * kJoinThreads, c = min(e / LANES, j.cols - 1);
                if (k0 + u >= j.count) continue;
                w[u][x] = reinterpret_cast<const float2*>(p)[c];
                v[u][x] = *reinterpret_cast<const float4*>(p + 2 * COLS + c * D + e % LANES * 4);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
        {
            if (k0 + u >= j.count) break;
#pragma unroll
            for (int x = 0; x < N; ++x)
            {
                const float top = fmaxf(M[x], w[u][x].x);
                const float f0 = M[x] == top ? 1.f : ex2(M[x] - top), f = w[u][x].x == top ? 1.f : ex2(w[u][x].x - top);
                L[x] = L[x] * f0 + f * w[u][x].y;
                o[x].x = o[x].x * f0 + f * v[u][x].x;
                o[x].y = o[x].y * f0 + f * v[u][x].y;
                o[x].z = o[x].z * f0 + f * v[u][x].z;
                o[x].w = o[x].w * f0 + f * v[u][x].w;
                M[x] = top;
            }
        }
    }
#pragma unroll
    for (int x = 0; x < N; ++x)
    {
        const int e = e0 + x * kJoinThreads, c = e / LANES;
        if (c >= j.cols) continue;
        const float inv = L[x] == 0.f ? 0.f : E::OUT / L[x];
        const float r[4] = {o[x].x * inv, o[x].y * inv, o[x].z * inv, o[x].w * inv};
        const int cc = j.col0 + c, rw = paged_row_of(a, cc);
        store_row<typename E::QT, 4>(a.out, (j.row0 + rw) * a.o_row_stride + (j.head * a.group + cc - rw * a.group) * a.o_head_stride + e % LANES * 4, r);
    }
}

}  // namespace hy
