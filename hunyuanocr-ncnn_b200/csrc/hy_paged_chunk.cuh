// Attention of many rows per sequence over the paged cache on the 5th-generation
// tensor cores (tcgen05), for bf16 rows over bf16, E4M3 and INT8 caches.
//
// An item is 256 columns (row, head of the group) of a KV head, as two tiles of
// 128, and the keys they see in blocks of 128; the items' blocks are shared out
// over the CTAs as in paged_split_kernel (one CTA per SM), and the parts of
// items that several CTAs share are joined by the same second kernel.
//
// Roles of a CTA's 16 warps, which meet at mbarriers only:
//   warps 0-3, 4-7: softmax of tile 0 and 1, one thread per column. The scores come
//     from tensor memory, the weights go back to it as the next product's operand;
//     the output is rescaled in tensor memory, and only when a column's maximum has
//     grown by more than 2^8 since it was last (the weights stay below 2^8);
//   warps 8-11: loads, and the walk over the items (the other roles read an item's
//     description from shared memory when its q is there). bf16 blocks arrive in the
//     128-byte-swizzled layout that serves K as the K-major operand of q k^T
//     and V as the MN-major operand of p v; 8-bit blocks arrive as codes in a
//     staging ring and are written to that layout as f16 (exact);
//   warp 12: one thread issues the products (13-15 make the warpgroup whole).
//     Tile 0's and 1's alternate, so that the tensor cores work on one tile while the
//     other's softmax runs: p v of block j, then q k^T of block j + 1, whose
//     scores take the place of the weights just used.
//
// Where pages hold a multiple of 16 rows, blocks are fetched by TMA, 16 rows of a
// page at a time (the window's start is rounded down to 16, masks do the rest);
// for other page sizes the loading warps copy row by row, from the very first key.
//
// 4 sequences of ~1012 rows over 6000-8192 bf16 keys (213 GFLOP): 243 us, 873 TFLOP/s, in a run of a few
// calls; 274 us, 777 TFLOP/s, back to back, where the power limit (990 W drawn) holds the SM clock at 1.74 GHz. The
// tensor cores are busy 45% of the time and the special-function units 45%: a tile's softmax
// and its products follow one another, and only two tiles fit tensor memory. Over 8-bit
// keys the softmax threads' products with the scales bound it (422 us; 16 softmax warps or 8 loading
// warps instead of 8 and 4 changed nothing: the windowed INT8 chunks take 236 and 240 us with them, 230 without). Pages of 24 rows
// instead of 32, copied by threads: 181 instead of 144 us (windowed chunks, bf16).
// ptxas spills 72 bytes a thread (BF16, 128 dimensions), 110 (BF16, 64), 118 and 130 (INT8 and E4M3, 128), 12 and 28
// (64); it does not say in which role.
//
// Tensor memory (512 columns): scores of the two tiles (128 each; the
// weights, 16 bits, in the upper 64 of them), outputs of the two tiles (128 each).
// Every wait is bounded and ends alike in a whole warp; a wait that gives up sets a status bit, the warp
// leaves its role, and the CTA runs on to free its tensor memory.
#pragma once

#include <cuda.h>

#include "hy_paged_attn.cuh"
#include "hy_tcgen05.cuh"

namespace hy {

template <typename CT_, int D_>
struct ChunkEngine {
    using QT = __nv_bfloat16;
    using CT = CT_;
    static constexpr int D = D_, COLS = 256, KEYS = 128;
    static constexpr bool F16 = kCodes<CT>;
    // f16 weights (times their values' scales) carry 2^6: below 2^(6 + 8 + 1), and rounded to 11 bits down to
    // 2^-20 of a row's largest, 2^-16 where one exponent stands for a block's scales; smaller ones lose bits, and below
    // 2^-27 nothing of them is left.
    static constexpr float OUT = F16 ? 1.f / 64.f : 1.f;
    static constexpr int RB = D * 2;                       // bytes of a row in operand layout
    static constexpr int TILE_B = 128 * RB;                // a block of K or V, a tile of q
    static constexpr int SLOTS = F16 ? 3 : 4;              // ring of K and V blocks
    static constexpr int CODES_B = 128 * D, STAGES = F16 ? 3 : 0;   // staging ring of 8-bit blocks
    static constexpr int Q_OFF = 0, RING_OFF = 2 * TILE_B, STAGE_OFF = RING_OFF + SLOTS * TILE_B;
    // Scales of the last 4 blocks: k, v times the weights' unit, exponent of v's (fp32, 128 each), in the order in
    // which the softmax threads take them: key 16 k + 8 e + 2 t + b at 16 k + 4 t + 2 e + b.
    static constexpr int SCALE_B = 3 * 128 * 4, SCALE_OFF = STAGE_OFF + STAGES * CODES_B;
    static constexpr int LIVE_OFF = SCALE_OFF + (F16 ? 4 * SCALE_B : 0);   // [4 blocks][4] words, a bit for every key
    static constexpr int EV_OFF = LIVE_OFF + 64;                           // [4 blocks][4] largest | smallest exponent << 16
    static constexpr int QS_OFF = EV_OFF + 64;                           // [256] 2^-k of a column's q
    static constexpr int ITEM_OFF = QS_OFF + 1024;                         // [2] ChunkItem
    static constexpr int BAR_OFF = ITEM_OFF + 2 * 64;
    static constexpr int SMEM = BAR_OFF + 320 + 1024;                      // + alignment of the base to 1024
    static_assert(SMEM <= 227 * 1024, "shared memory");
    static constexpr int S_COL = 0, O_COL = 256;           // tensor memory columns of tile 0; tile 1: + 128
};

// What the softmax and product roles need of an item.
struct ChunkItem {
    int row0, kv, n;            // the sequence
    int tile, head, cols;
    int sinks, lo, keys;        // virtual positions (PagedSpan)
    int b0, b1, tiles;          // this CTA's blocks [b0, b1) of tiles; b1 == b0: no more items
    int first;                  // the CTA's first item
    int lim[2];                 // where the blocks end that tile 0 / 1 sees something of, at most b1
    int last_cta;               // the CTA that has the item's last block
};

constexpr int kChunkThreads = 16 * 32;
constexpr int kChunkLoadWarp = 8, kChunkMmaWarp = 12;
// Registers a thread: 128 at launch; the 256 softmax threads take what the other 256 give up.
template <bool F16>
constexpr int kChunkRegsSoftmax = F16 ? 160 : 184;
template <bool F16>
constexpr int kChunkRegsOther = 2 * 128 - kChunkRegsSoftmax<F16>;
template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// True in one thread of the (converged) warp.
__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// Descriptor of an operand in the 128-byte-swizzled layout (layout type 2 at bits 61-63):
// rows of 128 bytes, eight rows to a 1024-byte atom.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo)
{
    return umma_desc(saddr, lbo, sbo) | (2ull << 61);
}
// Instruction descriptor, kind::f16: fp32 accumulator, A and B f16 (0) or bf16 (1), B
// MN-major when b_mn, N >> 3 at bit 17, M >> 4 at bit 24.
__host__ __device__ constexpr uint32_t idesc_f16(bool bf16, bool b_mn, int m, int n)
{
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t acc)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(acc)
        : "memory");
}
// 32 lanes x 32 consecutive 32-bit columns.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32_wait(uint32_t (&r)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(
            taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// 16 lanes x 32 columns as a warp's matrix fragments: register 4 k + j of thread t is (row t / 4 + 8 (j / 2),
// column 8 k + 2 (t % 4) + j % 2).
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_frag(uint32_t taddr, const uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// 16 lanes x 16 columns of packed pairs: register 2 k + j is (row t / 4 + 8 j, column 4 k + t % 4).
__device__ __forceinline__ void tmem_st_pairs(uint32_t taddr, const uint32_t (&r)[8])
{
    asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int c1, int c2, int c3, uint64_t* bar)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
        : "memory");
}
// Bounded waits of a whole (converged) warp: true in all its threads or in none, so that what comes next
// may be of the whole warp whichever way a wait ends.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status)
{
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, kPagedTimeout));
}
__device__ __forceinline__ bool warp_wait_spin(uint64_t* bar, uint32_t parity, int* status)
{
    return __all_sync(0xffffffffu, mbar_wait_spin(bar, parity, status, kPagedTimeout));
}
__device__ __forceinline__ bool warp_try_wait(uint64_t* bar, uint32_t parity)
{
    return __all_sync(0xffffffffu, mbar_try_wait(bar, parity));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Byte offset of 16-byte piece c of row r in a 128-row tile: 64 dimensions (128 bytes) to a
// block of 16 KB, pieces rotated by the row.
__device__ __forceinline__ uint32_t sw128_at(int r, int c)
{
    return static_cast<uint32_t>((c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// A CTA's walk over its share of the list of blocks.
template <int COLS, int TILE>
struct ItemWalk {
    SplitItem it;
    long long left;        // blocks of the share not yet walked over
    long long start;       // global index of the item's first block
    int units;             // (single) CTAs that share the item
    int b0, b1;            // blocks of the item that are this CTA's
    bool first, single;    // single: no second item
    int align;             // of the spans

    __device__ __forceinline__ bool open(const PagedAttnArgs& a, const SplitStart& st, int span_align)
    {
        align = span_align;
        left = (st.x1 - st.x0) * st.unit;
        single = st.unit > 1;
        first = true;
        if (left <= 0) return false;
        it.seq = st.seq;
        if (!paged_seq(a.b, it.seq, a.c.page_size, nullptr, it.q)) return false;
        long long in = st.in_seq;
        for (it.tile = 0;; ++it.tile)
        {
            it.w = paged_span(a, it.q, it.tile * COLS, COLS, align);
            it.tiles = split_tiles<TILE>(it.w.n);
            units = (it.tiles + st.unit - 1) / st.unit;
            if (in < static_cast<long long>(units) * a.c.kv_heads) break;
            if ((it.tile + 1) * COLS >= it.q.n * a.group) return false;   // (the arrays changed under the call)
            in -= static_cast<long long>(units) * a.c.kv_heads;
        }
        it.head = split_div(in, units);
        b0 = static_cast<int>(in - static_cast<long long>(it.head) * units) * st.unit;
        start = st.x0 - b0;
        set(a);
        return true;
    }
    // The CTA with the item's last block, where the item starts in CTA `cta`.
    __device__ __forceinline__ int last_cta(const SplitStart& st, int cta) const
    {
        return single ? cta + units - 1 : static_cast<int>((start + it.tiles - 1) / max(1ll, st.share));
    }
    __device__ __forceinline__ void set(const PagedAttnArgs& a)
    {
        b1 = static_cast<int>(min(static_cast<long long>(it.tiles), b0 + left));
        it.cols = min(COLS, it.q.n * a.group - it.tile * COLS);
    }
    __device__ __forceinline__ bool next(const PagedAttnArgs& a)
    {
        left -= b1 - b0;
        if (left <= 0 || single) return false;
        first = false;
        b0 = 0;
        start += it.tiles;
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
                if (it.seq >= a.b.num_seqs) return false;   // (the arrays changed under the call)
            }
            it.w = paged_span(a, it.q, it.tile * COLS, COLS, align);
            it.tiles = split_tiles<TILE>(it.w.n);
        }
        set(a);
        return true;
    }
    __device__ __forceinline__ bool complete() const { return b0 == 0 && b1 == it.tiles; }
    // Blocks of the item that tile i (0, 1) of its columns has anything to see in: [0, blocks).
    __device__ __forceinline__ int blocks(const PagedAttnArgs& a, int i) const
    {
        if (it.cols <= i * 128) return 0;
        const int last = min(it.cols, i * 128 + 128) - 1;
        const int p = it.q.kv - it.q.n + paged_row_of(a, it.tile * COLS + last);
        const int hi = p < 0 ? 0 : a.causal ? p + 1 : it.q.kv;
        // (virtual positions below that of key hi)
        const int n = hi <= it.w.sinks ? hi : hi <= it.w.lo ? it.w.sinks : it.w.sinks + hi - it.w.lo;
        return (n + TILE - 1) / TILE;
    }
};

// Largest of three; a NaN among them comes out.
__device__ __forceinline__ float max3_nan(float a, float b, float c)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Fetching by TMA: tensor maps of K and V over (dim, page, head, row), the last three in
// the order of their strides; where[i]: the coordinate (1..3) of row, head and page.
struct ChunkTma {
    CUtensorMap k, v;
    int on;
    int row_c, head_c, page_c;
};

template <typename CT, int D>
__global__ void __launch_bounds__(kChunkThreads, 1) paged_chunk_kernel(const PagedAttnArgs a, const __grid_constant__ ChunkTma tma)
{
    using E = ChunkEngine<CT, D>;
    using Walk = ItemWalk<256, 128>;
    constexpr bool F16 = E::F16;
    constexpr int SLOTS = E::SLOTS;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* const smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    const uint32_t sm = smem_u32(smem);
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + E::BAR_OFF);
    uint64_t* const kv_full = bars;               // [4] the block is in operand layout
    uint64_t* const kv_empty = kv_full + 4;       // [4] products that read it are done
    uint64_t* const st_full = kv_empty + 4;       // [3] codes are in the staging ring; bf16: [4] a warp's rows to be mended
    uint64_t* const st_empty = st_full + 4;       // [3] codes were read (4 warps)
    uint64_t* const q_full = st_empty + 3;        // the item's description is there, and (bf16) q (128)
    uint64_t* const q_empty = q_full + 1;         // products with q are done, the description was read (256)
    uint64_t* const s_full = q_empty + 1;         // [2] scores are there
    uint64_t* const p_full = s_full + 2;          // [2] weights are there (128), output rescaled
    uint64_t* const o_full = p_full + 2;          // [2] weights times values added
    uint64_t* const q_ready = o_full + 2;         // 8-bit caches: q is there (256)
    uint64_t* const done = q_ready + 1;           // every product is done
    uint64_t* const agreed = done + 1;            // [2] bf16: every thread of the tile looked for odd values (128)
    int* const pv_skip = reinterpret_cast<int*>(agreed + 2);   // [2] this block's product was taken by the softmax warps
    int* const odd_s = pv_skip + 2;                          // [2] the last block (1 + its number) in which a thread found some
    uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(odd_s + 2);
    float* const qscale = reinterpret_cast<float*>(smem + E::QS_OFF);
    ChunkItem* const items_s = reinterpret_cast<ChunkItem*>(smem + E::ITEM_OFF);
    volatile uint32_t* const live_w = reinterpret_cast<volatile uint32_t*>(smem + E::LIVE_OFF);
    volatile int* const ev_range = reinterpret_cast<volatile int*>(smem + E::EV_OFF);
    __shared__ long long scan[kChunkThreads / 32 + 1];
    static_assert(sizeof(ChunkItem) == 64, "item ring");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (warp == kChunkMmaWarp)
    {
        tmem_alloc(s_tmem, 512);
        tmem_relinquish();
    }
    if (tid == 0)
    {
        // (bf16 blocks by TMA: an arrival of each loading warp, with its own bytes; it also publishes the warp's
        // word of key-present bits)
        for (int i = 0; i < 4; ++i)
        {
            mbar_init(&kv_full[i], (!F16 && tma.on) ? 4 : 128);
            mbar_init(&kv_empty[i], 1);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&st_full[i], 1);
        for (int i = 0; i < 3; ++i) mbar_init(&st_empty[i], 4);
        mbar_init(q_full, 128);
        mbar_init(q_empty, 1 + 256);
        for (int i = 0; i < 2; ++i)
        {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 128);
            mbar_init(&o_full[i], 1);
            mbar_init(&agreed[i], 128);
            odd_s[i] = 0;
        }
        mbar_init(q_ready, 256);
        mbar_init(done, 1);
        fence_mbar_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    pdl_wait();
    pdl_launch();
    if (tid == 0) static_cast<PagedJoin*>(a.work)[blockIdx.x].count = 0;   // (rewritten below by the same thread)

    const int align = tma.on ? 16 : 1;   // (copied row by row, a block may start anywhere)
    const SplitStart st = split_start<256, 128, kChunkThreads>(a, scan, align);
    if (warp >= kChunkLoadWarp && warp < kChunkMmaWarp)
    {
        // ---------------- loads ----------------
        regs_dec<kChunkRegsOther<F16>>();
        const int lt = tid - kChunkLoadWarp * 32, lw = lt >> 5;
        Walk w;
        bool more = w.open(a, st, align);
        int n = 0;             // slots filled
        int blk = 0;           // blocks (index of the scale ring)
        int items = 0, mended = 0;
        int staged = 0;        // slots of the staging ring fetched
        bool ok_all = true;
        const bool leader = elect_one();
        for (;; ++items)
        {
            if (items) ok_all = ok_all && warp_wait(q_empty, (items - 1) & 1, a.c.status);
            if (lt == 0)
            {
                ChunkItem d;
                d.row0 = w.it.q.row0; d.kv = w.it.q.kv; d.n = w.it.q.n;
                d.tile = w.it.tile; d.head = w.it.head; d.cols = w.it.cols;
                d.sinks = w.it.w.sinks; d.lo = w.it.w.lo; d.keys = w.it.w.n;
                d.b0 = w.b0; d.b1 = w.b1; d.tiles = w.it.tiles;
                d.first = w.first;
                d.lim[0] = min(w.b1, w.blocks(a, 0));
                d.lim[1] = min(w.b1, w.blocks(a, 1));
                d.last_cta = w.last_cta(st, blockIdx.x);
                if (!more || !ok_all) d.b1 = d.b0;
                items_s[items & 1] = d;
            }
            if (!more || !ok_all)
            {
                mbar_arrive(q_full);
                break;
            }
            // q: rows of the two tiles, 256 columns, zero where there is no column.
            if constexpr (!F16)
            {
                constexpr int QP = E::RB / 16;   // 16-byte pieces of a row
#pragma unroll 4
                for (int x = lt; x < 256 * QP; x += 128)
                {
                    const int c = x / QP, p = x % QP;
                    const long long at = split_q_at(a, w.it, 256, min(c, w.it.cols - 1)) + p * 8;
                    cp_async16_zfill(sm + E::Q_OFF + (c >> 7) * E::TILE_B + sw128_at(c & 127, p),
                                     static_cast<const __nv_bfloat16*>(a.q) + at, c < w.it.cols);
                }
                cp_commit();
                cp_wait<0>();
            }
            // (8-bit caches: the softmax warps write q, as f16)
            fence_async_smem();
            mbar_arrive(q_full);

            const int* const table = a.b.table + w.it.seq * a.b.table_stride;
            auto find = [&](int b, int in_block, int& pg, int& row) {
                const int u = b * 128 + in_block;
                if (b >= w.b1 || u >= w.it.w.n) return;
                const int j = split_key(w.it, u), x = a.page_shift >= 0 ? j >> a.page_shift : j / a.c.page_size;
                row = j - x * a.c.page_size;
                pg = __ldg(table + x);
            };
            constexpr int CPR = D * static_cast<int>(sizeof(CT)) / 16;   // 16-byte pieces of a row in memory
            // Page and row: of this thread's key of a block, and (TMA) of the group of 16 keys 2 lw + lane % 2.
            int pg = 0, row = 0, gpg = 0, grow = 0;
            const int group_key = 32 * lw + (lane & 1) * 16;
            // This warp's two groups of a block by TMA, counted on `bar`.
            constexpr int WARP_BYTES = 32 * D * static_cast<int>(sizeof(CT));
            auto fetch = [&](int b, int kv, uint32_t dst, uint64_t* bar) {
                const bool ok = b * 128 + group_key < w.it.w.n && gpg >= 0 && gpg < a.c.num_pages;
                const int page = ok ? gpg : a.c.num_pages;   // (past the last page: zeros)
#pragma unroll
                for (int x = 0; x < 2; ++x)
                {
                    const int pgx = __shfl_sync(0xffffffffu, page, x), rwx = __shfl_sync(0xffffffffu, grow, x), g = 2 * lw + x;
                    const int c1 = tma.row_c == 1 ? rwx : tma.head_c == 1 ? w.it.head : pgx;
                    const int c2 = tma.row_c == 2 ? rwx : tma.head_c == 2 ? w.it.head : pgx;
                    const int c3 = tma.row_c == 3 ? rwx : tma.head_c == 3 ? w.it.head : pgx;
                    if (leader)
                    {
                        const CUtensorMap* const map = kv ? &tma.v : &tma.k;
                        tma_load_4d(dst + (F16 ? g * 16 * D : g * 2048), map, 0, c1, c2, c3, bar);
                        if constexpr (!F16 && D == 128) tma_load_4d(dst + 16384 + g * 2048, map, 64, c1, c2, c3, bar);
                    }
                }
                __syncwarp();
            };
            if constexpr (!F16)
            {
                if (tma.on)
                {
                    find(w.b0, group_key, gpg, grow);
                    for (int b = w.b0; b < w.b1 && ok_all; ++b, ++blk)
                    {
                        const int left = w.it.w.n - b * 128;   // keys from this block on
                        const bool page_ok = gpg >= 0 && gpg < a.c.num_pages;
                        const int cnt = lane < 2 ? min(max(left - group_key, 0), 16) : 0;
                        if (cnt && !page_ok) paged_status(a.c.status, kPagedBadPage);
                        const uint32_t bits = page_ok ? (1u << cnt) - 1u : 0u;
                        const uint32_t hi = __shfl_sync(0xffffffffu, bits, 1);
                        if (lane == 0) live_w[(blk & 3) * 4 + lw] = bits | (hi << 16);
                        __syncwarp();
                        // Rows behind the last key come along with its group; they may hold anything, and in V they
                        // become zeros before the products see them: the warp whose group it is arrives then.
                        const int mender = (left < 128 && (left & 15)) ? left >> 5 : -1;
#pragma unroll
                        for (int kv = 0; kv < 2; ++kv, ++n)
                        {
                            const int slot = n % SLOTS;
                            if (n >= SLOTS) ok_all = ok_all && warp_wait(&kv_empty[slot], (n / SLOTS - 1) & 1, a.c.status);
                            if (!ok_all) break;
                            const uint32_t dst = sm + E::RING_OFF + slot * E::TILE_B;
                            if (kv && mender == lw)
                            {
                                if (leader) mbar_arrive_expect_tx(&st_full[lw], WARP_BYTES);
                                __syncwarp();
                                fetch(b, kv, dst, &st_full[lw]);
                                ok_all = warp_wait(&st_full[lw], mended & 1, a.c.status);
                                ++mended;   // (of this warp)
                                if (!ok_all) break;
                                constexpr int QP = E::RB / 16;
                                for (int x = lane; x < (16 - (left & 15)) * QP; x += 32)
                                    *reinterpret_cast<uint4*>(smem + E::RING_OFF + slot * E::TILE_B + sw128_at(left + x / QP, x % QP)) = make_uint4(0, 0, 0, 0);
                                fence_async_smem();
                                __syncwarp();
                                if (leader) mbar_arrive(&kv_full[slot]);
                            }
                            else
                            {
                                if (leader) mbar_arrive_expect_tx(&kv_full[slot], WARP_BYTES);
                                __syncwarp();
                                fetch(b, kv, dst, &kv_full[slot]);
                            }
                        }
                        find(b + 1, group_key, gpg, grow);
                    }
                }
                else
                {
                    find(w.b0, lt, pg, row);
                    int sent = n;   // slots announced
                    auto drain = [&]() {
                        cp_wait<0>();
                        fence_async_smem();
                        for (; sent < n; ++sent) mbar_arrive(&kv_full[sent % SLOTS]);
                    };
                    for (int b = w.b0; b < w.b1 && ok_all; ++b, ++blk)
                    {
                        const bool there = b * 128 + lt < w.it.w.n;
                        const bool ok = there && pg >= 0 && pg < a.c.num_pages;
                        if (there && !ok) paged_status(a.c.status, kPagedBadPage);
                        const long long off = ok ? pg * a.c.page_stride + row * a.c.row_stride + w.it.head * a.c.head_stride : 0;
                        const uint32_t mask = __ballot_sync(0xffffffffu, ok);
                        if (lane == 0) live_w[(blk & 3) * 4 + lw] = mask;
                        find(b + 1, lt, pg, row);
#pragma unroll
                        for (int kv = 0; kv < 2; ++kv, ++n)
                        {
                            const int slot = n % SLOTS;
                            const CT* const base = static_cast<const CT*>(kv ? a.c.v : a.c.k);
                            if (n >= SLOTS && !warp_try_wait(&kv_empty[slot], (n / SLOTS - 1) & 1))
                            {
                                drain();   // what was fetched is on its way before this waits
                                ok_all = ok_all && warp_wait(&kv_empty[slot], (n / SLOTS - 1) & 1, a.c.status);
                                if (!ok_all) break;
                            }
                            const uint32_t dst = sm + E::RING_OFF + slot * E::TILE_B;
#pragma unroll 8
                            for (int x = 0; x < CPR; ++x)
                            {
                                const int idx = x * 32 + lane, r = idx / CPR, c = idx % CPR;
                                const long long o = __shfl_sync(0xffffffffu, off, r) + c * 8;
                                cp_async16_zfill(dst + sw128_at(lw * 32 + r, c), base + o, (mask >> r) & 1u);
                            }
                            cp_commit();
                            if (n - sent >= 2)
                            {
                                cp_wait<2>();
                                fence_async_smem();
                                mbar_arrive(&kv_full[sent % SLOTS]);
                                ++sent;
                            }
                        }
                    }
                    drain();
                }
            }
            else
            {
                // Codes to the staging ring two slots ahead, then to the operand ring as f16.
                const int n0 = n, n1 = n + 2 * (w.b1 - w.b0);
                int fb = w.b0;   // block of the next fetch
                if (tma.on) find(fb, group_key, gpg, grow);
                else find(fb, lt, pg, row);
                auto ahead = [&](int x) {   // fetch slot x
                    if (x < n1)
                    {
                        const int kv = (x - n0) & 1, sg = x % 3;
                        if (tma.on)
                        {
                            if (x >= 3) ok_all = ok_all && warp_wait(&st_empty[sg], (x / 3 - 1) & 1, a.c.status);
                            if (ok_all)
                            {
                                if (leader && lw == 0) mbar_arrive_expect_tx(&st_full[sg], 4 * WARP_BYTES);
                                fetch(fb, kv, sm + E::STAGE_OFF + sg * E::CODES_B, &st_full[sg]);
                                staged = x + 1;
                                if (kv) find(++fb, group_key, gpg, grow);
                            }
                        }
                        else
                        {
                            const bool ok = fb * 128 + lt < w.it.w.n && pg >= 0 && pg < a.c.num_pages;
                            const long long off = ok ? pg * a.c.page_stride + row * a.c.row_stride + w.it.head * a.c.head_stride : 0;
                            const uint32_t mask = __ballot_sync(0xffffffffu, ok);
                            const CT* const base = static_cast<const CT*>(kv ? a.c.v : a.c.k);
#pragma unroll
                            for (int y = 0; y < CPR; ++y)
                            {
                                const int idx = y * 32 + lane, r = idx / CPR, c = idx % CPR;
                                const long long o = __shfl_sync(0xffffffffu, off, r) + c * 16;
                                cp_async16_zfill(sm + E::STAGE_OFF + sg * E::CODES_B + (lw * 32 + r) * D + c * 16, base + o, (mask >> r) & 1u);
                            }
                            if (kv) find(++fb, lt, pg, row);
                        }
                    }
                    cp_commit();
                };
                // Page of this thread's key, for its scales: of block b, a block ahead of the scales themselves.
                int spg = 0, srow = 0;
                find(w.b0, lt, spg, srow);
                ahead(n0);
                ahead(n0 + 1);
                for (int b = w.b0; b < w.b1 && ok_all; ++b, ++blk)
                {
                    const bool there = b * 128 + lt < w.it.w.n;
                    const bool ok = there && spg >= 0 && spg < a.c.num_pages;
                    if (there && !ok) paged_status(a.c.status, kPagedBadPage);
                    const long long so = ok ? spg * a.c.s_page_stride + srow * a.c.s_row_stride + w.it.head * a.c.s_head_stride : 0;
                    const float ks = ok ? __ldg(a.c.k_scale + so) : 0.f, vs = ok ? __ldg(a.c.v_scale + so) : 0.f;
                    const uint32_t mask = __ballot_sync(0xffffffffu, ok);
                    find(b + 1, lt, spg, srow);
#pragma unroll 1
                    for (int kv = 0; kv < 2; ++kv, ++n)
                    {
                        const int slot = n % SLOTS, sg = n % 3;
                        ahead(n + 2);
                        if (tma.on) ok_all = ok_all && warp_wait(&st_full[sg], (n / 3) & 1, a.c.status);
                        else
                        {
                            cp_wait<2>();
                            __syncwarp();
                        }
                        if (n >= SLOTS) ok_all = ok_all && warp_wait(&kv_empty[slot], (n / SLOTS - 1) & 1, a.c.status);
                        if (!ok_all) break;
                        unsigned char* const dst = smem + E::RING_OFF + slot * E::TILE_B;
                        uint4 v[CPR];
#pragma unroll
                        for (int x = 0; x < CPR; ++x)
                        {
                            const int idx = x * 32 + lane, r = idx / CPR, c = idx % CPR;
                            v[x] = *reinterpret_cast<const uint4*>(smem + E::STAGE_OFF + sg * E::CODES_B + (lw * 32 + r) * D + c * 16);
                            if (!((mask >> r) & 1u)) v[x] = make_uint4(0, 0, 0, 0);   // (rows behind the last key)
                        }
#pragma unroll
                        for (int x = 0; x < CPR; ++x)
                        {
                            const int idx = x * 32 + lane, r = idx / CPR, c = idx % CPR, rr = lw * 32 + r;
                            *reinterpret_cast<uint4*>(dst + sw128_at(rr, 2 * c)) =
                                make_uint4(codes_f16<CT>(v[x].x), codes_f16<CT, true>(v[x].x), codes_f16<CT>(v[x].y), codes_f16<CT, true>(v[x].y));
                            *reinterpret_cast<uint4*>(dst + sw128_at(rr, 2 * c + 1)) =
                                make_uint4(codes_f16<CT>(v[x].z), codes_f16<CT, true>(v[x].z), codes_f16<CT>(v[x].w), codes_f16<CT, true>(v[x].w));
                        }
                        if (kv == 0)
                        {
                            // (entries of a block are written when the one four before it is long used)
                            float* const sc = reinterpret_cast<float*>(smem + E::SCALE_OFF + (blk & 3) * E::SCALE_B);
                            const int at = (lt >> 4) * 16 + ((lt >> 1) & 3) * 4 + ((lt >> 3) & 1) * 2 + (lt & 1);
                            const int ev = scale_exponent(vs);
                            sc[at] = ks;
                            sc[128 + at] = vs * 64.f;
                            sc[256 + at] = static_cast<float>(ev);
                            const int hi = __reduce_max_sync(0xffffffffu, ok ? ev : -100), lo = __reduce_min_sync(0xffffffffu, ok ? ev : 100);
                            if (lane == 0)
                            {
                                live_w[(blk & 3) * 4 + lw] = mask;
                                ev_range[(blk & 3) * 4 + lw] = (hi & 0xffff) | (lo << 16);
                            }
                        }
                        fence_async_smem();
                        mbar_arrive(&kv_full[slot]);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&st_empty[sg]);
                    }
                }
                cp_wait<0>();
            }
            more = w.next(a);
        }
        if (!ok_all && tma.on)
        {
            // After a wait that gave up: the block does not end before this warp's copies have landed (or as many
            // waits have given up again).
            if constexpr (F16)
                for (int x = max(0, staged - 3); x < staged; ++x) warp_wait(&st_full[x % 3], (x / 3) & 1, a.c.status);
            else
                for (int x = max(0, n - SLOTS); x < n; ++x) warp_wait(&kv_full[x % SLOTS], (x / SLOTS) & 1, a.c.status);
        }
    }
    else if (warp >= kChunkMmaWarp)
    {
        // ---------------- products ----------------
        regs_dec<kChunkRegsOther<F16>>();
        if (warp == kChunkMmaWarp)
        {
            // The whole warp walks, waits and computes addresses, so that they stay in uniform registers; one
            // thread issues. (With the whole loop under `lane == 0` an instruction took some 100 cycles to issue.)
            constexpr uint32_t ID_QK = idesc_f16(!F16, false, 128, 128), ID_PV = idesc_f16(!F16, true, 128, D);
            const bool leader = elect_one();
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            int nb = 0;   // blocks before this item
            int p_seen[2] = {0, 0};
            bool ok = true;
            auto qk = [&](int i, int blk) {
                const uint64_t qd = sw128_desc(sm + E::Q_OFF + i * E::TILE_B, 16, 1024);
                const uint64_t kd = sw128_desc(sm + E::RING_OFF + ((2 * blk) % SLOTS) * E::TILE_B, 16, 1024);
                if (leader)
                {
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks)
                    {
                        const uint64_t o = ((ks >> 2) * 16384 + (ks & 3) * 32) >> 4;
                        umma_f16_ss(tm + E::S_COL + i * 128, qd + o, kd + o, ID_QK, ks ? 1u : 0u);
                    }
                    umma_commit(&s_full[i]);
                }
                __syncwarp();
            };
            auto pv = [&](int i, int blk, bool add) {
                const uint64_t vd = sw128_desc(sm + E::RING_OFF + ((2 * blk + 1) % SLOTS) * E::TILE_B, 16384, 1024);
                if (leader)
                {
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks)
                        umma_f16_ts(tm + E::O_COL + i * 128, tm + E::S_COL + i * 128 + 64 + ks * 8, vd + ks * 128, ID_PV, (add || ks) ? 1u : 0u);
                }
                __syncwarp();
            };
            auto commit = [&](uint64_t* bar) {
                if (leader) umma_commit(bar);
                __syncwarp();
            };
            auto full = [&](int slot_n) {
                ok = ok && warp_wait_spin(&kv_full[slot_n % SLOTS], (slot_n / SLOTS) & 1, a.c.status);
                tc_fence_after();
            };
            for (int items = 0; ok; ++items)
            {
                ok = warp_wait_spin(q_full, items & 1, a.c.status);
                if (!ok) break;
                const ChunkItem it = items_s[items & 1];
                const int b0 = __shfl_sync(0xffffffffu, it.b0, 0), n_blk = __shfl_sync(0xffffffffu, it.b1, 0) - b0;
                const int lim[2] = {__shfl_sync(0xffffffffu, it.lim[0], 0), __shfl_sync(0xffffffffu, it.lim[1], 0)};
                if (n_blk <= 0) break;
                if constexpr (F16) ok = warp_wait_spin(q_ready, items & 1, a.c.status);
                full(2 * nb);
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (b0 < lim[i]) qk(i, nb);
                commit(&kv_empty[(2 * nb) % SLOTS]);
                if (n_blk == 1) commit(q_empty);
                for (int j = 0; j < n_blk && ok; ++j)
                {
                    const int blk = nb + j;
                    const bool more = j + 1 < n_blk;
                    bool v_there = false, k_there = false;
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                    {
                        if (ok && b0 + j < lim[i])
                        {
                            ok = warp_wait_spin(&p_full[i], p_seen[i] & 1, a.c.status);
                            ++p_seen[i];
                            if (!v_there) full(2 * blk + 1);
                            v_there = true;
                            tc_fence_after();
                            if (ok)
                            {
                                if (F16 || !*reinterpret_cast<volatile int*>(&pv_skip[i])) pv(i, blk, j > 0);
                                commit(&o_full[i]);
                            }
                        }
                        if (ok && more && b0 + j + 1 < lim[i])
                        {
                            if (!k_there) full(2 * blk + 2);
                            k_there = true;
                            if (ok) qk(i, blk + 1);
                        }
                    }
                    // (an item whose columns see nothing uses neither: their slots are free when they have arrived)
                    if (ok && !v_there) full(2 * blk + 1);
                    if (ok && more && !k_there) full(2 * blk + 2);
                    if (!ok) break;
                    commit(&kv_empty[(2 * blk + 1) % SLOTS]);
                    if (more) commit(&kv_empty[(2 * blk + 2) % SLOTS]);
                    if (j + 2 == n_blk) commit(q_empty);
                }
                nb += n_blk;
            }
            commit(done);   // nothing is in flight when the tensor memory is freed
            warp_wait_spin(done, 0, a.c.status);
        }
        __syncwarp();
    }
    else
    {
        // ---------------- softmax of tile i, one thread per column ----------------
        regs_inc<kChunkRegsSoftmax<F16>>();
        const int i = warp >> 2, c_in = tid & 127;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + E::S_COL + i * 128 + lanes, to = tmem + E::O_COL + i * 128 + lanes;
        int nb = 0, seen = 0;   // blocks of earlier items; blocks of this tile
        int masked = 0;         // bf16: those that not every column sees all of
        bool ok = true;
        for (int items = 0;; ++items)
        {
            ok = warp_wait(q_full, items & 1, a.c.status);
            if (!ok) break;
            const ChunkItem it = items_s[items & 1];
            const int c = i * 128 + c_in;
            mbar_arrive(q_empty);
            if (it.b1 == it.b0) break;
            const int lim = it.lim[i];
            const bool col = c < it.cols;
            const int p_0 = it.kv - it.n;
            // The tile's first and last positions.
            const int p_lo = p_0 + paged_row_of(a, it.tile * 256 + i * 128);
            const int p_hi = p_0 + paged_row_of(a, it.tile * 256 + min(it.cols, i * 128 + 128) - 1);
            auto key = [&](int u) { return u < it.sinks ? u : it.lo + u - it.sinks; };
            float m = -INFINITY, l = 0.f;
            // The keys that position pos sees of the 32 from virtual position u on, a bit each. They are (part of) the run
            // of sinks, then (part of) the window's: of either, the keys from the position's window on, and the sinks, up
            // to the position itself.
            auto see_word = [&](int pos, int u) {
                auto below = [](int x) { return x >= 32 ? 0xffffffffu : x <= 0 ? 0u : (1u << x) - 1u; };   // bits 0 .. x - 1
                const int split = it.sinks - u;   // keys that belong to the first run
                const int last = pos < 0 ? -1 : a.causal ? pos : it.kv - 1, from = a.window > 0 ? pos - a.window + 1 : 0;
                const int k1 = u, k2 = it.lo - split;   // key of bit 0 in the first and in the second run
                uint32_t in1 = below(last + 1 - k1), in2 = below(last + 1 - k2);
                if (a.window > 0)
                {
                    in1 &= ~below(from - k1) | below(a.sinks - k1);
                    in2 &= ~below(from - k2) | below(a.sinks - k2);
                }
                const uint32_t one = below(split);
                return (in1 & one) | (in2 & ~one);
            };
            // Every column of the tile sees every key of block u0, whose bits are `vis`.
            auto sees_all = [&](int u0, const uint32_t (&vis)[4]) {
                const int j_first = key(u0), j_last = key(min(u0 + 127, it.keys - 1));
                return (vis[0] & vis[1] & vis[2] & vis[3]) == 0xffffffffu && p_lo >= 0 &&
                       (!a.causal || (j_last <= p_lo && (a.window == 0 || j_first > p_hi - a.window || j_last < a.sinks)));
            };
            // Of values that are in the fragments' threads, this thread's column's.
            auto of_row = [&](const float (&v)[4]) {
                float x[4];
#pragma unroll
                for (int f = 0; f < 4; ++f) x[f] = __shfl_sync(0xffffffffu, v[f], (lane & 7) * 4);
                const int f = lane >> 3;
                return f == 0 ? x[0] : f == 1 ? x[1] : f == 2 ? x[2] : x[3];
            };
            if constexpr (!F16)
            {
            const float fac = a.scale_log2;
            const int p = col ? p_0 + paged_row_of(a, it.tile * 256 + c) : -1;
            for (int b = it.b0; b < lim && ok; ++b, ++seen)
            {
                const int blk = nb + b - it.b0, ring = blk & 3, vslot = (2 * blk + 1) % SLOTS;
                // (the values' barrier tells that the block's scales and bits are there too, and its slot
                // cannot be filled anew before this tile's weights are out)
                ok = warp_wait(&kv_full[vslot], ((2 * blk + 1) / SLOTS) & 1, a.c.status) &&
                     warp_wait(&s_full[i], seen & 1, a.c.status);
                if (!ok) break;
                tc_fence_after();
                uint32_t r[128];   // scores, then (packed) weights
                uint32_t(&r0)[32] = *reinterpret_cast<uint32_t(*)[32]>(r);
                uint32_t(&r1)[32] = *reinterpret_cast<uint32_t(*)[32]>(r + 32);
                uint32_t(&r2)[32] = *reinterpret_cast<uint32_t(*)[32]>(r + 64);
                uint32_t(&r3)[32] = *reinterpret_cast<uint32_t(*)[32]>(r + 96);
                tmem_ld32(ts, r0);
                tmem_ld32(ts + 32, r1);
                tmem_ld32(ts + 64, r2);
                tmem_ld32(ts + 96, r3);
                const int u0 = b * 128;
                uint32_t vis[4];   // what the column sees, a bit per key
                {
                    const uint4 x = lds128(sm + E::LIVE_OFF + ring * 16);
                    vis[0] = x.x; vis[1] = x.y; vis[2] = x.z; vis[3] = x.w;
                }
                const bool whole = sees_all(u0, vis);
                bool odd = false;
                tmem_ld32_wait(r0);
                tmem_ld32_wait(r1);
                tmem_ld32_wait(r2);
                tmem_ld32_wait(r3);
                if (!whole)
                {
#pragma unroll
                    for (int x = 0; x < 4; ++x) vis[x] &= see_word(p, u0 + 32 * x);
#pragma unroll
                    for (int e = 0; e < 128; ++e)
                        if (!((vis[e >> 5] >> (e & 31)) & 1u)) r[e] = 0xff800000u;   // -inf
                    {
                        // 0 times an infinity or NaN is NaN, so a block that some column must not see all of and
                        // that holds such values is not for the tensor cores.
                        uint32_t bad = 0;
                        for (int x = c_in; x < E::TILE_B / 16; x += 128)
                        {
                            const uint4 q = lds128(sm + E::RING_OFF + vslot * E::TILE_B + x * 16);
                            const uint32_t ws[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) bad |= (ws[e] & 0x7f800000u) == 0x7f800000u || (ws[e] & 0x7f80u) == 0x7f80u;
                        }
                        // (the mark of this block stands until the tile's weights are out)
                        if (bad) *reinterpret_cast<volatile int*>(&odd_s[i]) = seen + 1;
                        mbar_arrive(&agreed[i]);
                        ok = warp_wait(&agreed[i], masked & 1, a.c.status);
                        ++masked;
                        if (!ok) break;
                        odd = *reinterpret_cast<volatile int*>(&odd_s[i]) == seen + 1;
                    }
                }
                float top;
                {
                    float t0 = -INFINITY, t1 = -INFINITY, t2 = -INFINITY, t3 = -INFINITY;
                    auto z = [&](int e) { return __uint_as_float(r[e]); };
#pragma unroll
                    for (int e = 0; e < 128; e += 8)
                    {
                        t0 = max3_nan(t0, z(e), z(e + 1));
                        t1 = max3_nan(t1, z(e + 2), z(e + 3));
                        t2 = max3_nan(t2, z(e + 4), z(e + 5));
                        t3 = max3_nan(t3, z(e + 6), z(e + 7));
                    }
                    top = max3_nan(max3_nan(t0, t1, t2), t3, t3);
                    top *= fac;
                }
                if (top == INFINITY) top = __int_as_float(0x7fffffff);   // inf - inf
                // A new reference only where the maximum has grown by more than 2^8 (or there was none); a NaN becomes one.
                const bool grow = !(top <= m + 8.f) && !(top == -INFINITY);
                float corr = 1.f;
                if (grow)
                {
                    corr = ex2(m - top);
                    l *= corr;
                    m = top;
                }
                if (b > it.b0 && __any_sync(0xffffffffu, grow))
                {
                    ok = warp_wait(&o_full[i], (seen - 1) & 1, a.c.status);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int x = 0; x < D / 16; ++x)
                    {
                        uint32_t o[16];
                        tmem_ld16(to + 16 * x, o);
                        tmem_ld_wait(o);
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                        tmem_st16(to + 16 * x, o);
                    }
                }
                const float mm = m == -INFINITY ? 0.f : m;
                const uint64_t fac2 = f2(fac, fac), mm2 = f2(-mm, -mm);
                uint64_t sum0 = 0, sum1 = 0;   // (pairs of zeros)
#pragma unroll
                for (int e = 0; e < 64; ++e)
                {
                    float w0, w1;
                    f2_get(f2_fma(f2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), fac2, mm2), w0, w1);
                    w0 = ex2(w0);
                    w1 = ex2(w1);
                    if (e & 1) sum1 = f2_add(sum1, f2(w0, w1));
                    else sum0 = f2_add(sum0, f2(w0, w1));
                    r[e] = pack_bf16(w0, w1);
                    if (e == 31) tmem_st32(ts + 64, *reinterpret_cast<uint32_t(*)[32]>(r));
                }
                tmem_st32(ts + 96, *reinterpret_cast<uint32_t(*)[32]>(r + 32));
                float s0, s1, s2, s3;
                f2_get(sum0, s0, s1);
                f2_get(sum1, s2, s3);
                l += (s0 + s1) + (s2 + s3);
                tmem_st_wait();
                {
                    if (odd)
                    {
                        // o += p v, key by key, for what the column sees.
                        if (b > it.b0) ok = warp_wait(&o_full[i], (seen - 1) & 1, a.c.status);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t vbase = sm + E::RING_OFF + vslot * E::TILE_B;
                        auto vis_at = [&](int x) { return x == 0 ? vis[0] : x == 1 ? vis[1] : x == 2 ? vis[2] : vis[3]; };
#pragma unroll 1
                        for (int x = 0; x < D / 16; ++x)
                        {
                            uint32_t o[16];
                            tmem_ld16(to + 16 * x, o);
                            tmem_ld_wait(o);
                            if (b == it.b0)
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] = 0;
#pragma unroll 1
                            for (int k = 0; k < 128; ++k)
                            {
                                uint32_t pw;   // the word of keys k and k ^ 1
                                asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(pw) : "r"(ts + 64 + (k >> 1)) : "memory");
                                asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(pw)::"memory");
                                const float pk = __uint_as_float((k & 1) ? pw & 0xFFFF0000u : pw << 16);
                                if ((vis_at(k >> 5) >> (k & 31)) & 1u)
                                {
#pragma unroll
                                    for (int e = 0; e < 2; ++e)
                                    {
                                        const uint4 v = lds128(vbase + sw128_at(k, 2 * x + e));
                                        const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                                        for (int y = 0; y < 4; ++y)
                                        {
                                            uint32_t& o0 = o[8 * e + 2 * y];
                                            uint32_t& o1 = o[8 * e + 2 * y + 1];
                                            o0 = __float_as_uint(fmaf(pk, __uint_as_float(vw[y] << 16), __uint_as_float(o0)));
                                            o1 = __float_as_uint(fmaf(pk, __uint_as_float(vw[y] & 0xFFFF0000u), __uint_as_float(o1)));
                                        }
                                    }
                                }
                                __syncwarp();
                            }
                            tmem_st16(to + 16 * x, o);
                        }
                        tmem_st_wait();
                    }
                    if (c_in == 0) *reinterpret_cast<volatile int*>(&pv_skip[i]) = odd;
                }
                tc_fence_before();
                mbar_arrive(&p_full[i]);
            }
            }
            else
            {
                // 8-bit caches: every score and weight meets its key's scales. With a column to a thread those
                // would be 128 loads a thread and array - more shared-memory time than the products take -, so
                // the scores are taken as matrix fragments: a thread has 32 keys of 4 columns, 8 f + lane / 4.
                {
                    // q of this thread's column as f16, times the power of two that brings its largest magnitude to
                    // [2^14, 2^15). (This tile's products with the last item's q are done: their scores were read.)
                    constexpr int QP = E::RB / 16;   // 16-byte pieces of a row
                    const uint4* const src = reinterpret_cast<const uint4*>(
                        static_cast<const __nv_bfloat16*>(a.q) + (it.row0 + paged_row_of(a, it.tile * 256 + min(c, it.cols - 1))) * a.q_row_stride +
                        (it.head * a.group + it.tile * 256 + min(c, it.cols - 1) - paged_row_of(a, it.tile * 256 + min(c, it.cols - 1)) * a.group) * a.q_head_stride);
                    uint4 raw[QP];
                    uint32_t top = 0;
#pragma unroll
                    for (int x = 0; x < QP; ++x) raw[x] = __ldg(src + x);
#pragma unroll
                    for (int x = 0; x < QP; ++x)
                    {
                        if (!col) raw[x] = make_uint4(0, 0, 0, 0);
                        top = __vmaxu2(top, __vmaxu2(__vmaxu2(raw[x].x & 0x7fff7fffu, raw[x].y & 0x7fff7fffu),
                                                     __vmaxu2(raw[x].z & 0x7fff7fffu, raw[x].w & 0x7fff7fffu)));
                    }
                    top = max(top << 16, top & 0x7fff0000u);
                    const uint32_t down = (min(max(top >> 23, 16u), 254u) - 14u) << 23;
                    const float up = __uint_as_float((254u << 23) - down);
                    qscale[c] = __uint_as_float(down);
#pragma unroll
                    for (int x = 0; x < QP; ++x)
                    {
                        auto half = [&](uint32_t w) { return pack_f16(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xFFFF0000u) * up); };
                        *reinterpret_cast<uint4*>(smem + E::Q_OFF + i * E::TILE_B + sw128_at(c_in, x)) =
                            make_uint4(half(raw[x].x), half(raw[x].y), half(raw[x].z), half(raw[x].w));
                    }
                    fence_async_smem();
                    mbar_arrive(q_ready);
                    __syncwarp();
                }
                const int c_0 = i * 128 + (warp & 3) * 32 + (lane >> 2);   // column of f = 0
                float fac[4], mf[4], lf[4];
                int pos[4];
#pragma unroll
                for (int f = 0; f < 4; ++f)
                {
                    fac[f] = fmaxf(a.scale_log2 * qscale[c_0 + 8 * f], 1e-45f);   // (0 times a masked -inf is NaN)
                    pos[f] = c_0 + 8 * f < it.cols ? p_0 + paged_row_of(a, it.tile * 256 + c_0 + 8 * f) : -1;
                    mf[f] = -INFINITY;
                    lf[f] = 0.f;
                }
                for (int b = it.b0; b < lim && ok; ++b, ++seen)
                {
                    const int blk = nb + b - it.b0, ring = blk & 3, vslot = (2 * blk + 1) % SLOTS;
                    ok = warp_wait(&kv_full[vslot], ((2 * blk + 1) / SLOTS) & 1, a.c.status) &&
                         warp_wait(&s_full[i], seen & 1, a.c.status);
                    if (!ok) break;
                    tc_fence_after();
                    const float4* const sc = reinterpret_cast<const float4*>(smem + E::SCALE_OFF + ring * E::SCALE_B) + (lane & 3);
                    uint32_t live[4];
                    int ev_hi, ev_lo;
                    {
                        const uint4 x = lds128(sm + E::LIVE_OFF + ring * 16);
                        live[0] = x.x; live[1] = x.y; live[2] = x.z; live[3] = x.w;
                        const uint4 y = lds128(sm + E::EV_OFF + ring * 16);
                        ev_hi = max(max(static_cast<short>(y.x), static_cast<short>(y.y)), max(static_cast<short>(y.z), static_cast<short>(y.w)));
                        ev_lo = min(min(static_cast<int>(y.x) >> 16, static_cast<int>(y.y) >> 16), min(static_cast<int>(y.z) >> 16, static_cast<int>(y.w) >> 16));
                    }
                    const bool whole = sees_all(b * 128, live);
                    // The reference takes in the exponents of the values' scales. Where they are close, the block's
                    // largest serves every key; it must be of keys that the columns see. Weights are then smaller by up to
                    // 2^4: with 2^12 a row of 16000 light keys beside a heavy one lost them all.
                    const bool tight = whole && ev_hi - ev_lo <= 4;
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    // First pass, 32 keys at a time (loops, not straight code: four roles' instructions compete for the
                    // instruction cache): scores times their keys' scales, masked, back to tensor memory; the maxima.
                    uint32_t r[2][16], next[2][16];   // [h]: columns f = 2 h, 2 h + 1
                    auto fetch = [&](int x, uint32_t (&to)[2][16]) {
                        tmem_ld_frag(ts + 32 * x, to[0]);
                        tmem_ld_frag(ts + 32 * x + (16u << 16), to[1]);
                    };
                    auto take = [&]() {
                        tmem_ld_wait(next[0]);
                        tmem_ld_wait(next[1]);
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int e = 0; e < 16; ++e) r[h][e] = next[h][e];
                    };
                    fetch(0, next);
                    take();
#pragma unroll 1
                    for (int x = 0; x < 4; ++x)
                    {
                        fetch(min(x + 1, 3), next);   // (the last round's is not used)
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                        {
                            const float4 ks = sc[4 * (2 * x + k)];
#pragma unroll
                            for (int e = 0; e < 2; ++e)
#pragma unroll
                                for (int f = 0; f < 4; ++f)
                                {
                                    const int at = 8 * k + 4 * e + 2 * (f & 1);
                                    uint32_t(&q)[16] = r[f >> 1];
                                    float u, v;
                                    f2_get(f2_mul(f2(__uint_as_float(q[at]), __uint_as_float(q[at + 1])), e ? f2(ks.z, ks.w) : f2(ks.x, ks.y)), u, v);
                                    q[at] = __float_as_uint(u);
                                    q[at + 1] = __float_as_uint(v);
                                }
                        }
                        if (!whole)
                        {
                            const uint32_t here = x == 0 ? live[0] : x == 1 ? live[1] : x == 2 ? live[2] : live[3];
#pragma unroll
                            for (int f = 0; f < 4; ++f)
                            {
                                const uint32_t v = (here & see_word(pos[f], b * 128 + 32 * x)) >> (2 * (lane & 3));
#pragma unroll
                                for (int e = 0; e < 8; ++e)   // key 8 (e / 2) + e % 2 + 2 (lane % 4)
                                    if (!((v >> (8 * (e >> 1) + (e & 1))) & 1u)) r[f >> 1][4 * (e >> 1) + 2 * (f & 1) + (e & 1)] = 0xff800000u;   // -inf
                            }
                        }
                        if (tight)
                        {
#pragma unroll
                            for (int k = 0; k < 4; ++k)
#pragma unroll
                                for (int f = 0; f < 4; ++f)
                                    top[f] = max3_nan(top[f], __uint_as_float(r[f >> 1][4 * k + 2 * (f & 1)]), __uint_as_float(r[f >> 1][4 * k + 2 * (f & 1) + 1]));
                        }
                        else
                        {
#pragma unroll
                            for (int k = 0; k < 2; ++k)
                            {
                                const float4 ev = sc[64 + 4 * (2 * x + k)];
#pragma unroll
                                for (int e = 0; e < 2; ++e)
#pragma unroll
                                    for (int f = 0; f < 4; ++f)
                                    {
                                        const int at = 8 * k + 4 * e + 2 * (f & 1);
                                        top[f] = max3_nan(top[f], fmaf(__uint_as_float(r[f >> 1][at]), fac[f], e ? ev.z : ev.x),
                                                          fmaf(__uint_as_float(r[f >> 1][at + 1]), fac[f], e ? ev.w : ev.y));
                                    }
                            }
                        }
                        tmem_st_frag(ts + 32 * x, r[0]);
                        tmem_st_frag(ts + 32 * x + (16u << 16), r[1]);
                        take();
                    }
                    if (tight)
#pragma unroll
                        for (int f = 0; f < 4; ++f) top[f] = fmaf(top[f], fac[f], static_cast<float>(ev_hi));
                    tmem_st_wait();
                    fetch(3, next);
                    take();
                    bool grew = false;
                    float corr[4], mm[4];
                    uint64_t sum[4];
#pragma unroll
                    for (int f = 0; f < 4; ++f)
                    {
                        top[f] = max3_nan(top[f], __shfl_xor_sync(0xffffffffu, top[f], 1), top[f]);
                        top[f] = max3_nan(top[f], __shfl_xor_sync(0xffffffffu, top[f], 2), top[f]);
                        if (top[f] == INFINITY) top[f] = __int_as_float(0x7fffffff);   // inf - inf
                        const bool grow = !(top[f] <= mf[f] + 8.f) && !(top[f] == -INFINITY);
                        corr[f] = 1.f;
                        if (grow)
                        {
                            corr[f] = ex2(mf[f] - top[f]);
                            lf[f] *= corr[f];
                            mf[f] = top[f];
                            grew = true;
                        }
                        mm[f] = mf[f] == -INFINITY ? 0.f : -mf[f];
                        sum[f] = 0;
                    }
                    if (b > it.b0 && __any_sync(0xffffffffu, grew))
                    {
                        ok = warp_wait(&o_full[i], (seen - 1) & 1, a.c.status);
                        if (!ok) break;
                        tc_fence_after();
                        const float mine = of_row(corr);
#pragma unroll 1
                        for (int x = 0; x < D / 16; ++x)
                        {
                            uint32_t o[16];
                            tmem_ld16(to + 16 * x, o);
                            tmem_ld_wait(o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * mine);
                            tmem_st16(to + 16 * x, o);
                        }
                    }
                    // Second pass, from the last keys on: a chunk's weights take the place of scores that are done.
                    auto weights = [&](auto plain) {
                        constexpr bool PLAIN = decltype(plain)::value;   // the columns see the whole block
#pragma unroll 1
                        for (int x = 3; x >= 0; --x)
                        {
                            fetch(max(x - 1, 0), next);
                            uint32_t out[2][8];
#pragma unroll
                            for (int k = 0; k < 2; ++k)
                            {
                                const float4 vs = sc[32 + 4 * (2 * x + k)];
#pragma unroll
                                for (int e = 0; e < 2; ++e)
#pragma unroll
                                    for (int f = 0; f < 4; ++f)
                                    {
                                        const int at = 8 * k + 4 * e + 2 * (f & 1);
                                        const uint32_t s0 = r[f >> 1][at], s1 = r[f >> 1][at + 1];
                                        uint64_t y = f2_fma(f2(__uint_as_float(s0), __uint_as_float(s1)), f2(fac[f], fac[f]), f2(mm[f], mm[f]));
                                        float w0, w1;
                                        f2_get(y, w0, w1);
                                        y = f2(ex2(w0), ex2(w1));
                                        sum[f] = f2_add(sum[f], y);
                                        f2_get(f2_mul(y, e ? f2(vs.z, vs.w) : f2(vs.x, vs.y)), w0, w1);
                                        if constexpr (!PLAIN)
                                        {
                                            // (a scale of NaN must not meet a weight of zero that stands for "not seen")
                                            if (s0 == 0xff800000u) w0 = 0.f;
                                            if (s1 == 0xff800000u) w1 = 0.f;
                                        }
                                        out[f >> 1][4 * k + 2 * e + (f & 1)] = pack_f16(w0, w1);
                                    }
                            }
                            tmem_st_pairs(ts + 64 + 16 * x, out[0]);
                            tmem_st_pairs(ts + 64 + 16 * x + (16u << 16), out[1]);
                            take();
                        }
                    };
                    if (whole) weights(std::true_type{});
                    else weights(std::false_type{});
#pragma unroll
                    for (int f = 0; f < 4; ++f)
                    {
                        float x, y;
                        f2_get(sum[f], x, y);
                        lf[f] += x + y;
                    }
                    tmem_st_wait();
                    tc_fence_before();
                    mbar_arrive(&p_full[i]);
                }
#pragma unroll
                for (int f = 0; f < 4; ++f)
                {
                    lf[f] += __shfl_xor_sync(0xffffffffu, lf[f], 1);
                    lf[f] += __shfl_xor_sync(0xffffffffu, lf[f], 2);
                }
                m = of_row(mf);
                l = of_row(lf);
            }
            if (!ok) break;
            // ---- the item's output, or this CTA's part of it ----
            const bool any = lim > it.b0;
            if (any)
            {
                ok = warp_wait(&o_full[i], (seen - 1) & 1, a.c.status);
                if (!ok) break;
                tc_fence_after();
            }
            const bool complete = it.b0 == 0 && it.b1 == it.tiles;
            const int part_slot = 2 * blockIdx.x + (it.first ? 0 : 1);
            float* const part = reinterpret_cast<float*>(static_cast<unsigned char*>(a.work) + kSplitDescBytes) +
                                static_cast<long long>(part_slot) * (256 * (D + 2));
            const float inv = l == 0.f ? 0.f : E::OUT / l;
            if (i * 128 < it.cols)
            {
                if (col && !complete) reinterpret_cast<float2*>(part)[c] = make_float2(m, l);
                if (col && complete && a.lse) paged_put_lse(a, it.row0, it.head, it.tile * 256 + c, m, l);
                const int cc = it.tile * 256 + c, rw = paged_row_of(a, cc);
                const long long at = (it.row0 + rw) * a.o_row_stride + (it.head * a.group + cc - rw * a.group) * a.o_head_stride;
#pragma unroll 1
                for (int x = 0; x < D / 32; ++x)
                {
                    uint32_t o[32];
                    tmem_ld32(to + 32 * x, o);
                    tmem_ld32_wait(o);
                    if (col)
                    {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                        {
                            float v[8];
#pragma unroll
                            for (int y = 0; y < 8; ++y) v[y] = any ? __uint_as_float(o[8 * e + y]) : 0.f;
                            if (complete)
                            {
#pragma unroll
                                for (int y = 0; y < 8; ++y) v[y] *= inv;
                                store_row<__nv_bfloat16, 8>(a.out, at + 32 * x + 8 * e, v);
                            }
                            else
                            {
                                float4* const d = reinterpret_cast<float4*>(part + 512 + c * D + 32 * x + 8 * e);
                                d[0] = make_float4(v[0], v[1], v[2], v[3]);
                                d[1] = make_float4(v[4], v[5], v[6], v[7]);
                            }
                        }
                    }
                    __syncwarp();
                }
                tc_fence_before();
            }
            if (tid == 0 && !complete && it.b0 == 0)
            {
                PagedJoin d;
                d.count = it.last_cta - static_cast<int>(blockIdx.x) + 1;
                d.first_slot = part_slot;
                d.first_cta = blockIdx.x;
                d.row0 = it.row0;
                d.col0 = it.tile * 256;
                d.cols = it.cols;
                d.head = it.head;
                d.pad = 0;
                static_cast<PagedJoin*>(a.work)[blockIdx.x] = d;
            }
            nb += it.b1 - it.b0;
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == kChunkMmaWarp)
    {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace hy
