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
//   warps 8-11: loads. Every thread looks up the page of one key of a block;
//     rows go to shared memory by cp.async (bf16) or through registers as f16 (8-bit codes, exact),
//     in the 128-byte-swizzled layout that serves K as the K-major operand of
//     q k^T and V as the MN-major operand of p v;
//   warp 12: one thread issues the products (13-15 make the warpgroup whole). Tile 0's and 1's alternate, so
//     that the tensor cores work on one tile while the other's softmax runs:
//     p v of block j, then q k^T of block j + 1, whose scores take the place of the weights just used.
//
// Tensor memory (512 columns): scores of the two tiles (128 each; the
// weights, 16 bits, in the upper 64 of them), outputs of the two tiles (128 each).
// Every wait is bounded; a wait that gives up sets a status bit, and the CTA
// runs on to free its tensor memory.
#pragma once

#include "hy_paged_attn.cuh"
#include "hy_tcgen05.cuh"

namespace hy {

template <typename CT_, int D_>
struct ChunkEngine {
    using QT = __nv_bfloat16;
    using CT = CT_;
    static constexpr int D = D_, COLS = 256, KEYS = 128;
    static constexpr bool F16 = kCodes<CT>;
    // f16 weights carry 2^6: below 2^(6 + 8 + 1), and exact to 11 bits down to 2^-20 of the largest.
    static constexpr float OUT = F16 ? 1.f / 64.f : 1.f;
    static constexpr int RB = D * 2;                       // bytes of a row in shared memory
    static constexpr int TILE_B = 128 * RB;                // a block of K or V, a tile of q
    static constexpr int SLOTS = 4;                        // ring of K and V blocks
    static constexpr int Q_OFF = 0, RING_OFF = 2 * TILE_B;
    // Scales of the last 4 blocks: k, v times the weights' unit, exponent of v's (fp32, 128 each).
    static constexpr int SCALE_B = 3 * 128 * 4, SCALE_OFF = RING_OFF + SLOTS * TILE_B;
    static constexpr int LIVE_OFF = SCALE_OFF + (F16 ? 4 * SCALE_B : 0);   // [4 blocks][4] words, a bit for every key
    static constexpr int QS_OFF = LIVE_OFF + 64;                      // [256] 2^-k of a column's q
    static constexpr int BAR_OFF = QS_OFF + 1024;
    static constexpr int SMEM = BAR_OFF + 256 + 1024;                 // + alignment of the base to 1024
    static constexpr int S_COL = 0, O_COL = 256;           // tensor memory columns of tile 0; tile 1: + 128
};

constexpr int kChunkThreads = 16 * 32;
constexpr int kChunkLoadWarp = 8, kChunkMmaWarp = 12;
// Registers a thread: 128 at launch; 256 softmax threads take 184, the other 256 keep 72
// (184 + 72 = 2 x 128: what one half gives up is what the other asks for).
constexpr int kChunkRegsSoftmax = 184, kChunkRegsOther = 72;
static_assert(kChunkRegsSoftmax + kChunkRegsOther == 2 * 128, "registers");
template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

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
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Byte offset of 16-byte piece c of row r in a 128-row tile: 64 dimensions (128 bytes) to a
// block of 16 KB, pieces rotated by the row.
__device__ __forceinline__ uint32_t sw128_at(int r, int c)
{
    return static_cast<uint32_t>((c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// A CTA's walk over its share of the list of blocks; every role keeps its own.
template <int COLS, int TILE>
struct ItemWalk {
    SplitItem it;
    long long left;        // blocks of the share not yet walked over
    long long start;       // global index of the item's first block
    int b0, b1;            // blocks of the item that are this CTA's
    bool first;

    __device__ __forceinline__ bool open(const PagedAttnArgs& a, const SplitStart& st)
    {
        left = st.x1 - st.x0;
        first = true;
        if (left <= 0) return false;
        it.seq = st.seq;
        if (!paged_seq(a.b, it.seq, a.c.page_size, nullptr, it.q)) return false;
        long long in = st.in_seq;
        for (it.tile = 0;; ++it.tile)
        {
            it.w = paged_span(a, it.q, it.tile * COLS, COLS);
            it.tiles = split_tiles<TILE>(it.w.n);
            if (in < static_cast<long long>(it.tiles) * a.c.kv_heads) break;
            if ((it.tile + 1) * COLS >= it.q.n * a.group) return false;   // (the arrays changed under the call)
            in -= static_cast<long long>(it.tiles) * a.c.kv_heads;
        }
        it.head = static_cast<int>(in / it.tiles);
        b0 = static_cast<int>(in - static_cast<long long>(it.head) * it.tiles);
        start = st.x0 - b0;
        set(a);
        return true;
    }
    __device__ __forceinline__ void set(const PagedAttnArgs& a)
    {
        b1 = static_cast<int>(min(static_cast<long long>(it.tiles), b0 + left));
        it.cols = min(COLS, it.q.n * a.group - it.tile * COLS);
    }
    __device__ __forceinline__ bool next(const PagedAttnArgs& a)
    {
        left -= b1 - b0;
        if (left <= 0) return false;
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
            it.w = paged_span(a, it.q, it.tile * COLS, COLS);
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
        const int p = it.q.kv - it.q.n + (it.tile * COLS + last) / a.group;
        const int hi = p < 0 ? 0 : a.causal ? p + 1 : it.q.kv;
        // (virtual positions below that of key hi)
        const int n = hi <= it.w.sinks ? hi : hi <= it.w.lo ? it.w.sinks : it.w.sinks + hi - it.w.lo;
        return (n + TILE - 1) / TILE;
    }
};

template <typename CT, int D>
__global__ void __launch_bounds__(kChunkThreads, 1) paged_chunk_kernel(const PagedAttnArgs a)
{
    using E = ChunkEngine<CT, D>;
    using Walk = ItemWalk<256, 128>;
    constexpr bool F16 = E::F16;
    constexpr int SLOTS = E::SLOTS;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* const smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    const uint32_t sm = smem_u32(smem);
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + E::BAR_OFF);
    uint64_t* const kv_full = bars;               // [SLOTS] 128 loading threads
    uint64_t* const kv_empty = kv_full + SLOTS;   // [SLOTS] products that read it are done
    uint64_t* const q_full = kv_empty + SLOTS;    // 128
    uint64_t* const q_empty = q_full + 1;         // products with q are done, qscale was read (256)
    uint64_t* const s_full = q_empty + 1;         // [2] scores are there
    uint64_t* const p_full = s_full + 2;          // [2] weights are there (128), output rescaled
    uint64_t* const o_full = p_full + 2;          // [2] weights times values added
    uint64_t* const done = o_full + 2;            // every product is done
    int* const pv_skip = reinterpret_cast<int*>(done + 1);   // [2] this block's product was taken by the softmax warps
    uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(pv_skip + 2);
    float* const qscale = reinterpret_cast<float*>(smem + E::QS_OFF);
    volatile uint32_t* const live_w = reinterpret_cast<volatile uint32_t*>(smem + E::LIVE_OFF);
    __shared__ long long scan[kChunkThreads / 32 + 1];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (warp == kChunkMmaWarp)
    {
        tmem_alloc(s_tmem, 512);
        tmem_relinquish();
    }
    if (tid == 0)
    {
        for (int i = 0; i < SLOTS; ++i)
        {
            mbar_init(&kv_full[i], 128);
            mbar_init(&kv_empty[i], 1);
        }
        mbar_init(q_full, 128);
        mbar_init(q_empty, 1 + 256);
        mbar_init(done, 1);
        for (int i = 0; i < 2; ++i)
        {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 128);
            mbar_init(&o_full[i], 1);
        }
        fence_mbar_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    pdl_wait();
    pdl_launch();
    const SplitStart st = split_start<256, 128, kChunkThreads>(a, scan);
    PagedJoin* const desc = static_cast<PagedJoin*>(a.work) + blockIdx.x;
    if (tid == 0) desc->count = 0;   // (rewritten below by the same thread)

    Walk w;
    bool more = w.open(a, st);
    if (warp >= kChunkLoadWarp && warp < kChunkMmaWarp)
    {
        // ---------------- loads ----------------
        regs_dec<kChunkRegsOther>();
        const int lt = tid - kChunkLoadWarp * 32, lw = lt >> 5;
        int n = 0;             // slots filled
        int blk = 0;           // blocks loaded (index of the scale ring)
        int items = 0;
        bool ok_all = true;
        for (; more && ok_all; more = w.next(a), ++items)
        {
            // q: rows of the two tiles, 256 columns, zero where there is no column.
            if (items) ok_all = mbar_wait(q_empty, (items - 1) & 1, a.c.status, kPagedTimeout);
            constexpr int QP = E::RB / 16;   // 16-byte pieces of a row
            if constexpr (!F16)
            {
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
            else
            {
                // As f16, times the power of two that brings the column's largest magnitude to [2^14, 2^15).
                constexpr int LPC = QP;   // lanes of a column
                for (int x = lt; x < 256 * QP; x += 128)
                {
                    const int c = x / QP, p = x % QP;
                    float v[8];
                    load_row<__nv_bfloat16, 8>(a.q, split_q_at(a, w.it, 256, min(c, w.it.cols - 1)) + p * 8, v);
                    uint32_t m = 0;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                    {
                        if (c >= w.it.cols) v[e] = 0.f;
                        m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
                    }
#pragma unroll
                    for (int o = 1; o < LPC; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
                    const uint32_t down = (min(max(m >> 23, 16u), 254u) - 14u) << 23;
                    const float up = __uint_as_float((254u << 23) - down);
                    if (p == 0) qscale[c] = __uint_as_float(down);
                    *reinterpret_cast<uint4*>(smem + E::Q_OFF + (c >> 7) * E::TILE_B + sw128_at(c & 127, p)) =
                        make_uint4(pack_f16(v[0] * up, v[1] * up), pack_f16(v[2] * up, v[3] * up),
                                   pack_f16(v[4] * up, v[5] * up), pack_f16(v[6] * up, v[7] * up));
                }
            }
            fence_async_smem();
            mbar_arrive(q_full);

            const int* const table = a.b.table + w.it.seq * a.b.table_stride;
            int pg_next = 0, row_next = 0;
            auto look_up = [&](int b) {
                const int u = b * 128 + lt;
                if (b >= w.b1 || u >= w.it.w.n) return;
                const int j = split_key(w.it, u), x = a.page_shift >= 0 ? j >> a.page_shift : j / a.c.page_size;
                row_next = j - x * a.c.page_size;
                pg_next = __ldg(table + x);
            };
            look_up(w.b0);
            const int n_item = n;
            for (int b = w.b0; b < w.b1 && ok_all; ++b, ++blk)
            {
                const bool there = b * 128 + lt < w.it.w.n;
                const bool ok = there && pg_next >= 0 && pg_next < a.c.num_pages;
                if (there && !ok) paged_status(a.c.status, kPagedBadPage);
                const long long off = ok ? pg_next * a.c.page_stride + row_next * a.c.row_stride + w.it.head * a.c.head_stride : 0;
                const uint32_t mask = __ballot_sync(0xffffffffu, ok);
                if constexpr (F16)
                {
                    const long long so = ok ? pg_next * a.c.s_page_stride + row_next * a.c.s_row_stride + w.it.head * a.c.s_head_stride : 0;
                    float* const sc = reinterpret_cast<float*>(smem + E::SCALE_OFF + (blk & 3) * E::SCALE_B);
                    const float vs = ok ? __ldg(a.c.v_scale + so) : 0.f;
                    sc[lt] = ok ? __ldg(a.c.k_scale + so) : 0.f;
                    sc[128 + lt] = vs * 64.f;
                    sc[256 + lt] = static_cast<float>(min(max(static_cast<int>(__float_as_uint(vs) >> 23) - 127, -100), 100));
                }
                if (lane == 0) live_w[(blk & 3) * 4 + lw] = mask;
                look_up(b + 1);
#pragma unroll
                for (int kv = 0; kv < 2; ++kv, ++n)
                {
                    const int slot = n % SLOTS;
                    const CT* const base = static_cast<const CT*>(kv ? a.c.v : a.c.k);
                    constexpr int CPR = D * static_cast<int>(sizeof(CT)) / 16;   // pieces of a row in memory
                    if constexpr (!F16)
                    {
                        if (n >= SLOTS) ok_all = ok_all && mbar_wait(&kv_empty[slot], (n / SLOTS - 1) & 1, a.c.status, kPagedTimeout);
                        const uint32_t dst = sm + E::RING_OFF + slot * E::TILE_B;
#pragma unroll
                        for (int x = 0; x < CPR; ++x)
                        {
                            const int idx = x * 32 + lane, r = idx / CPR, c = idx % CPR;
                            const long long o = __shfl_sync(0xffffffffu, off, r) + c * 8;
                            cp_async16_zfill(dst + sw128_at(lw * 32 + r, c), base + o, (mask >> r) & 1u);
                        }
                        cp_commit();
                        if (n - n_item >= 2)
                        {
                            cp_wait<2>();
                            fence_async_smem();
                            mbar_arrive(&kv_full[(n - 2) % SLOTS]);
                        }
                    }
                    else
                    {
                        uint4 v[CPR];
#pragma unroll
                        for (int x = 0; x < CPR; ++x)
                        {
                            const int idx = x * 32 + lane, r = idx / CPR, c = idx % CPR;
                            const long long o = __shfl_sync(0xffffffffu, off, r) + c * 16;
                            v[x] = ((mask >> r) & 1u) ? __ldg(reinterpret_cast<const uint4*>(base + o)) : make_uint4(0, 0, 0, 0);
                        }
                        if (n >= SLOTS) ok_all = ok_all && mbar_wait(&kv_empty[slot], (n / SLOTS - 1) & 1, a.c.status, kPagedTimeout);
                        unsigned char* const dst = smem + E::RING_OFF + slot * E::TILE_B;
#pragma unroll
                        for (int x = 0; x < CPR; ++x)
                        {
                            const int idx = x * 32 + lane, r = lw * 32 + idx / CPR, c = idx % CPR;
                            *reinterpret_cast<uint4*>(dst + sw128_at(r, 2 * c)) =
                                make_uint4(codes_f16<CT>(v[x].x), codes_f16<CT>(v[x].x >> 16), codes_f16<CT>(v[x].y), codes_f16<CT>(v[x].y >> 16));
                            *reinterpret_cast<uint4*>(dst + sw128_at(r, 2 * c + 1)) =
                                make_uint4(codes_f16<CT>(v[x].z), codes_f16<CT>(v[x].z >> 16), codes_f16<CT>(v[x].w), codes_f16<CT>(v[x].w >> 16));
                        }
                        fence_async_smem();
                        mbar_arrive(&kv_full[slot]);
                    }
                }
            }
            if constexpr (!F16)
            {
                cp_wait<0>();
                fence_async_smem();
                for (int x = max(n_item, n - 2); x < n; ++x) mbar_arrive(&kv_full[x % SLOTS]);
            }
        }
        cp_wait<0>();
    }
    else if (warp >= kChunkMmaWarp)
    {
        // ---------------- products ----------------
        regs_dec<kChunkRegsOther>();
        if (warp == kChunkMmaWarp && lane == 0)
        {
            constexpr uint32_t ID_QK = idesc_f16(!F16, false, 128, 128), ID_PV = idesc_f16(!F16, true, 128, D);
            int nb = 0, items = 0;   // blocks before this item
            int p_seen[2] = {0, 0};
            bool ok = true;
            auto qk = [&](int i, int blk) {
                const uint32_t q = sm + E::Q_OFF + i * E::TILE_B, k = sm + E::RING_OFF + ((2 * blk) % SLOTS) * E::TILE_B;
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                {
                    const uint32_t o = (ks >> 2) * 16384 + (ks & 3) * 32;
                    umma_f16_ss(tmem + E::S_COL + i * 128, sw128_desc(q + o, 16, 1024), sw128_desc(k + o, 16, 1024), ID_QK, ks ? 1u : 0u);
                }
                umma_commit(&s_full[i]);
            };
            auto pv = [&](int i, int blk, bool add) {
                const uint32_t v = sm + E::RING_OFF + ((2 * blk + 1) % SLOTS) * E::TILE_B;
#pragma unroll
                for (int ks = 0; ks < 8; ++ks)
                    umma_f16_ts(tmem + E::O_COL + i * 128, tmem + E::S_COL + i * 128 + 64 + ks * 8,
                                sw128_desc(v + ks * 2048, 16384, 1024), ID_PV, (add || ks) ? 1u : 0u);
            };
            auto full = [&](int slot_n) {
                ok = ok && mbar_wait_spin(&kv_full[slot_n % SLOTS], (slot_n / SLOTS) & 1, a.c.status, kPagedTimeout);
                tc_fence_after();
            };
            for (; more && ok; more = w.next(a), ++items)
            {
                const int lim[2] = {min(w.b1, w.blocks(a, 0)), min(w.b1, w.blocks(a, 1))};
                const int n_blk = w.b1 - w.b0;
                ok = ok && mbar_wait_spin(q_full, items & 1, a.c.status, kPagedTimeout);
                full(2 * nb);
                if (!ok) break;
                for (int i = 0; i < 2; ++i)
                    if (w.b0 < lim[i]) qk(i, nb);
                umma_commit(&kv_empty[(2 * nb) % SLOTS]);
                if (n_blk == 1) umma_commit(q_empty);
                for (int j = 0; j < n_blk && ok; ++j)
                {
                    const int blk = nb + j;
                    full(2 * blk + 1);
                    if (j + 1 < n_blk) full(2 * blk + 2);
                    for (int i = 0; i < 2 && ok; ++i)
                    {
                        if (w.b0 + j < lim[i])
                        {
                            ok = mbar_wait_spin(&p_full[i], p_seen[i] & 1, a.c.status, kPagedTimeout);
                            ++p_seen[i];
                            if (!ok) break;
                            tc_fence_after();
                            if (F16 || !*reinterpret_cast<volatile int*>(&pv_skip[i])) pv(i, blk, j > 0);
                            umma_commit(&o_full[i]);
                        }
                        if (j + 1 < n_blk && w.b0 + j + 1 < lim[i]) qk(i, blk + 1);
                    }
                    if (!ok) break;
                    umma_commit(&kv_empty[(2 * blk + 1) % SLOTS]);
                    if (j + 1 < n_blk) umma_commit(&kv_empty[(2 * blk + 2) % SLOTS]);
                    if (j + 2 == n_blk) umma_commit(q_empty);
                }
                nb += n_blk;
            }
            umma_commit(done);   // nothing is in flight when the tensor memory is freed
            mbar_wait_spin(done, 0, a.c.status, kPagedTimeout);
        }
        __syncwarp();
    }
    else
    {
        // ---------------- softmax of tile i, one thread per column ----------------
        regs_inc<kChunkRegsSoftmax>();
        const int i = warp >> 2, c_in = tid & 127;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + E::S_COL + i * 128 + lanes, to = tmem + E::O_COL + i * 128 + lanes;
        float* const parts = reinterpret_cast<float*>(static_cast<unsigned char*>(a.work) + kSplitDescBytes);
        int nb = 0, seen = 0, items = 0;   // blocks of earlier items; blocks of this tile; items
        bool ok = true;
        for (; more && ok; more = w.next(a), ++items)
        {
            const int lim = min(w.b1, w.blocks(a, i));
            const int c = i * 128 + c_in, cc = w.it.tile * 256 + c, rw = cc / a.group;
            const bool col = c < w.it.cols;
            const int p = col ? w.it.q.kv - w.it.q.n + rw : -1;
            // The tile's first and last positions.
            const int p_lo = w.it.q.kv - w.it.q.n + (w.it.tile * 256 + i * 128) / a.group;
            const int p_hi = w.it.q.kv - w.it.q.n + (w.it.tile * 256 + min(w.it.cols, i * 128 + 128) - 1) / a.group;
            ok = mbar_wait(q_full, items & 1, a.c.status, kPagedTimeout);
            if (!ok) break;
            const float fac = F16 ? a.scale_log2 * qscale[c] : a.scale_log2;
            mbar_arrive(q_empty);
            float m = -INFINITY, l = 0.f;
            for (int b = w.b0; b < lim && ok; ++b, ++seen)
            {
                const int blk = nb + b - w.b0, ring = blk & 3, vslot = (2 * blk + 1) % SLOTS;
                // (the values' barrier tells that the block's scales and bits are there too, and its slot
                // cannot be filled anew before this tile's weights are out)
                ok = mbar_wait(&kv_full[vslot], ((2 * blk + 1) / SLOTS) & 1, a.c.status, kPagedTimeout) &&
                     mbar_wait(&s_full[i], seen & 1, a.c.status, kPagedTimeout);
                if (!ok) break;
                tc_fence_after();
                const float4* const sc = reinterpret_cast<const float4*>(smem + E::SCALE_OFF + ring * E::SCALE_B);
                const int u0 = b * 128, j_first = split_key(w.it, u0), j_last = split_key(w.it, min(u0 + 127, w.it.w.n - 1));
                uint32_t vis[4];   // what the column sees, a bit per key
#pragma unroll
                for (int x = 0; x < 4; ++x) vis[x] = live_w[ring * 4 + x];
                const bool whole = (vis[0] & vis[1] & vis[2] & vis[3]) == 0xffffffffu && p_lo >= 0 &&
                                   (!a.causal || (j_last <= p_lo && (a.window == 0 || j_first > p_hi - a.window || j_last < a.sinks)));
                bool odd = false;
                if (!whole)
                {
                    if (u0 >= w.it.w.sinks)   // one run of keys
                    {
                        const int hi = p < 0 ? -1 : a.causal ? min(p - j_first, 127) : 127;
                        const int lo = a.window > 0 && p - a.window + 1 > j_first ? p - a.window + 1 - j_first : 0;
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                        {
                            const int h = hi - 32 * x, f = lo - 32 * x;
                            uint32_t in = h >= 31 ? 0xffffffffu : h < 0 ? 0u : (2u << h) - 1u;
                            in &= f <= 0 ? 0xffffffffu : f > 31 ? 0u : 0xffffffffu << f;
                            // (keys below the window may still be sinks)
                            const int s = min(a.sinks - j_first - 32 * x, 32);
                            if (a.window > 0 && s > 0) in |= (s >= 32 ? 0xffffffffu : (1u << s) - 1u) & (h >= 31 ? 0xffffffffu : h < 0 ? 0u : (2u << h) - 1u);
                            vis[x] &= in;
                        }
                    }
                    else
                    {
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                        {
                            uint32_t in = 0;
#pragma unroll 1
                            for (int y = 0; y < 32; ++y)
                                in |= (paged_sees(a, p, split_key(w.it, u0 + 32 * x + y)) ? 1u : 0u) << y;
                            vis[x] &= in;
                        }
                    }
                    if constexpr (!F16)
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
                        uint32_t any;
                        asm volatile(
                            "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                            : "=r"(any)
                            : "r"(bad), "r"(1 + i)
                            : "memory");
                        odd = any != 0;
                    }
                }
                // Scores of chunk x (32 keys), in units that `fac` makes powers of two; -inf where not seen.
                auto scores = [&](int x, uint32_t (&r)[32]) {
                    if constexpr (F16)
                    {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                        {
                            const float4 k = sc[x * 8 + e];
                            r[4 * e] = __float_as_uint(__uint_as_float(r[4 * e]) * k.x);
                            r[4 * e + 1] = __float_as_uint(__uint_as_float(r[4 * e + 1]) * k.y);
                            r[4 * e + 2] = __float_as_uint(__uint_as_float(r[4 * e + 2]) * k.z);
                            r[4 * e + 3] = __float_as_uint(__uint_as_float(r[4 * e + 3]) * k.w);
                        }
                    }
                    if (!whole)
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!((vis[x] >> e) & 1u)) r[e] = 0xff800000u;
                };
                auto top_of = [&](int x, const uint32_t (&r)[32]) {
                    float t0 = -INFINITY, t1 = -INFINITY, t2 = -INFINITY, t3 = -INFINITY;
                    if constexpr (F16)
                    {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                        {
                            const float4 v = sc[64 + x * 8 + e];
                            t0 = fmaxf(t0, fmaf(__uint_as_float(r[4 * e]), fac, v.x));
                            t1 = fmaxf(t1, fmaf(__uint_as_float(r[4 * e + 1]), fac, v.y));
                            t2 = fmaxf(t2, fmaf(__uint_as_float(r[4 * e + 2]), fac, v.z));
                            t3 = fmaxf(t3, fmaf(__uint_as_float(r[4 * e + 3]), fac, v.w));
                        }
                        return fmaxf(fmaxf(t0, t1), fmaxf(t2, t3));
                    }
                    else
                    {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                        {
                            t0 = fmaxf(t0, __uint_as_float(r[4 * e]));
                            t1 = fmaxf(t1, __uint_as_float(r[4 * e + 1]));
                            t2 = fmaxf(t2, __uint_as_float(r[4 * e + 2]));
                            t3 = fmaxf(t3, __uint_as_float(r[4 * e + 3]));
                        }
                        return fmaxf(fmaxf(t0, t1), fmaxf(t2, t3));
                    }
                };
                uint32_t ra[32], rb[32];
                tmem_ld32(ts, ra);
                tmem_ld32(ts + 32, rb);
                tmem_ld32_wait(ra);
                tmem_ld32_wait(rb);
                scores(0, ra);
                scores(1, rb);
                float top = fmaxf(top_of(0, ra), top_of(1, rb));
                tmem_ld32(ts + 64, ra);
                tmem_ld32(ts + 96, rb);
                tmem_ld32_wait(ra);
                tmem_ld32_wait(rb);
                scores(2, ra);
                scores(3, rb);
                top = fmaxf(top, fmaxf(top_of(2, ra), top_of(3, rb)));
                if constexpr (!F16) top = top == -INFINITY ? top : top * fac;
                // A new reference only where the maximum has grown by more than 2^8 (or there was none).
                const bool grow = top > m + 8.f || (m == -INFINITY && top > m);
                float corr = 1.f;
                if (grow)
                {
                    corr = ex2(m - top);
                    l *= corr;
                    m = top;
                }
                if (b > w.b0 && __any_sync(0xffffffffu, grow))
                {
                    ok = mbar_wait(&o_full[i], (seen - 1) & 1, a.c.status, kPagedTimeout);
                    tc_fence_after();
#pragma unroll 1
                    for (int x = 0; x < D / 32; ++x)
                    {
                        uint32_t o[32];
                        tmem_ld32(to + 32 * x, o);
                        tmem_ld32_wait(o);
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                        tmem_st32(to + 32 * x, o);
                    }
                }
                const float mm = m == -INFINITY ? 0.f : m;
                float l0 = 0.f, l1 = 0.f;
                // The weights of chunks x and x + 1 as the next product's operand, 32 words.
                auto weights = [&](int x, const uint32_t (&r0)[32], const uint32_t (&r1)[32]) {
                    uint32_t out[32];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                        {
                            const uint32_t s0 = h ? r1[2 * e] : r0[2 * e], s1 = h ? r1[2 * e + 1] : r0[2 * e + 1];
                            float w0 = ex2(fmaf(__uint_as_float(s0), fac, -mm)), w1 = ex2(fmaf(__uint_as_float(s1), fac, -mm));
                            l0 += w0;
                            l1 += w1;
                            if constexpr (F16)
                            {
                                const float2 v = reinterpret_cast<const float2*>(sc)[64 + (x + h) * 16 + e];
                                w0 *= v.x;
                                w1 *= v.y;
                                // (a scale of NaN must not meet a weight of zero that stands for "not seen")
                                if (!whole && !((vis[x + h] >> (2 * e)) & 1u)) w0 = 0.f;
                                if (!whole && !((vis[x + h] >> (2 * e + 1)) & 1u)) w1 = 0.f;
                                out[16 * h + e] = pack_f16(w0, w1);
                            }
                            else
                            {
                                out[16 * h + e] = pack_bf16(w0, w1);
                            }
                        }
                    tmem_st32(ts + 64 + 16 * x, out);
                };
                weights(2, ra, rb);   // over scores that are in registers
                tmem_ld32(ts, ra);
                tmem_ld32(ts + 32, rb);
                tmem_ld32_wait(ra);
                tmem_ld32_wait(rb);
                scores(0, ra);
                scores(1, rb);
                weights(0, ra, rb);
                l += l0 + l1;
                tmem_st_wait();
                if constexpr (!F16)
                {
                    if (odd)
                    {
                        // o += p v, key by key, for what the column sees.
                        if (b > w.b0) ok = ok && mbar_wait(&o_full[i], (seen - 1) & 1, a.c.status, kPagedTimeout);
                        tc_fence_after();
                        const uint32_t vbase = sm + E::RING_OFF + vslot * E::TILE_B;
                        auto vis_at = [&](int x) { return x == 0 ? vis[0] : x == 1 ? vis[1] : x == 2 ? vis[2] : vis[3]; };
#pragma unroll 1
                        for (int x = 0; x < D / 32; ++x)
                        {
                            uint32_t o[32];
                            tmem_ld32(to + 32 * x, o);
                            tmem_ld32_wait(o);
                            if (b == w.b0)
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] = 0;
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
                                    for (int e = 0; e < 4; ++e)
                                    {
                                        const uint4 v = lds128(vbase + sw128_at(k, 4 * x + e));
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
                            tmem_st32(to + 32 * x, o);
                        }
                        tmem_st_wait();
                    }
                    if (c_in == 0) *reinterpret_cast<volatile int*>(&pv_skip[i]) = odd;
                }
                tc_fence_before();
                mbar_arrive(&p_full[i]);
            }
            if (!ok) break;
            // ---- the item's output, or this CTA's part of it ----
            const bool any = lim > w.b0;
            if (any)
            {
                ok = mbar_wait(&o_full[i], (seen - 1) & 1, a.c.status, kPagedTimeout);
                if (!ok) break;
                tc_fence_after();
            }
            const bool complete = w.complete();
            const int part_slot = 2 * blockIdx.x + (w.first ? 0 : 1);
            float* const part = parts + static_cast<long long>(part_slot) * (256 * (D + 2));
            const float inv = l == 0.f ? 0.f : E::OUT / l;
            if (i * 128 < w.it.cols)
            {
                if (col && !complete) reinterpret_cast<float2*>(part)[c] = make_float2(m, l);
                const long long at = (w.it.q.row0 + rw) * a.o_row_stride + (w.it.head * a.group + cc - rw * a.group) * a.o_head_stride;
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
            if (tid == 0 && !complete && w.b0 == 0)
            {
                const long long x_last = w.start + w.it.tiles - 1;   // global index of the item's last block
                PagedJoin d;
                d.count = static_cast<int>(x_last / st.share) - static_cast<int>(blockIdx.x) + 1;
                d.first_slot = part_slot;
                d.first_cta = blockIdx.x;
                d.row0 = w.it.q.row0;
                d.col0 = w.it.tile * 256;
                d.cols = w.it.cols;
                d.head = w.it.head;
                d.pad = 0;
                *desc = d;
            }
            nb += w.b1 - w.b0;
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
