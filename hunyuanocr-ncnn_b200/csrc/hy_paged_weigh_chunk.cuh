// Attention weights of cached positions (hy_paged_weigh.cuh) for many bf16 rows over
// bf16, E4M3 and INT8 caches, on the 5th-generation tensor cores (tcgen05).
//
// An item is one or two blocks of 128 keys of a (sequence, KV head), which stay in shared
// memory as the A operand while the columns that see any of them stream by in tiles of 128, the B
// operand: S^T = K Q^T comes to lie in tensor memory with a key to a lane, so that a thread has
// all scores of its key, one tile after another, and nothing is ever reduced across
// threads. Two blocks to an item, so that q is fetched (from L2) half as often.
//
// Roles of a CTA's 21 warps, which meet at mbarriers only:
//   warps 0-15: exponentials and sums. Four warps (128 keys) take the even tiles for block 0, four for block 1, and
//     eight the odd tiles; the two sums of a key are added up when its columns are through. So a tile's hand-over and
//     products (some 1600 cycles) run under the other tile's exponentials (2048).
//   warps 16-19: loads, and the walk over the list. Each fetches a quarter of an item's keys (8-bit ones become
//     bf16 on the way, exactly), and every fourth tile of q alone, so that four fetches are under way: by TMA
//     where a tile is a box of q (group a power of two), else by cp.async, column by column;
//   warp 20: the products.
//
// Tensor memory: scores of two tiles for each of the two blocks, 4 x 128 columns, so that
// the products of a tile run under the exponentials of the one before. 4 sequences of ~1012 rows over 6000-8192 bf16
// keys (111 GFLOP): 163 us, 683 TFLOP/s; the special-function units are busy 70% of the time (101 us of exponentials),
// the tensor cores 35%, and the CTAs' shares, whole blocks, differ by 12%.  Every wait is bounded, as in hy_paged_chunk.cuh.
#pragma once

#include <climits>

#include "hy_paged_chunk.cuh"
#include "hy_paged_weigh.cuh"

namespace hy {

constexpr int kWeighChunkWarps = 21;
constexpr int kWeighChunkThreads = kWeighChunkWarps * 32;
constexpr int kWeighLoadWarp = 16, kWeighMmaWarp = 20;

template <typename CT_, int D_>
struct WeighChunk {
    using CT = CT_;
    static constexpr int D = D_, KEYS = 128, COLS = 128;
    static constexpr int RB = D * 2, BLOCK_B = 128 * RB;             // bytes of a row and of 128 rows in operand layout
    static constexpr int K_OFF = 0;                                  // [2 blocks]
    static constexpr int Q_OFF = 2 * BLOCK_B;                        // [4 tiles]
    static constexpr int INFO_OFF = Q_OFF + 4 * BLOCK_B;             // [8 tiles] -lse and position of 128 columns
    static constexpr int INFO_B = 2 * 128 * 4;
    static constexpr int ITEM_OFF = INFO_OFF + 8 * INFO_B;           // WeighItem
    static constexpr int PART_OFF = ITEM_OFF + 64;                   // [2 items][2 blocks][128] sums of the odd tiles
    static constexpr int BAR_OFF = PART_OFF + 4 * 128 * 4;
    static constexpr int SMEM = BAR_OFF + 256 + 1024;                // + alignment of the base to 1024
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

// Tensor map of q over (dim, head, row), a box being 64 dimensions of a tile's 128 columns.
struct WeighTma {
    CUtensorMap q;
    int on;
};

// What the other roles need of an item.
struct WeighItem {
    int seq, head, row0, kv, n;
    int keys, sinks, lo;     // virtual positions (PagedSpan)
    int block, blocks;       // first block, 1 or 2; 0: no more items
    int c0, tiles;           // the columns: tiles of 128 from column c0 on
    int pad[4];
};

// Bytes to come in the barrier's phase, without an arrival.
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes)
{
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// One arrival for a whole warp, after what all its lanes did. (256 arrivals of threads at one barrier are taken one after
// another, and cost a tile more than its products.)
__device__ __forceinline__ void warp_arrive(uint64_t* bar)
{
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// The columns that see any of the keys of blocks [b, b + blocks) of a sequence: from column c0 on, in tiles of 128.
__device__ __forceinline__ void weigh_columns(const PagedAttnArgs& a, const PagedSeq& q, const PagedSpan& w, int b, int blocks, int& c0, int& tiles)
{
    const int u_first = b * 128, u_last = min((b + blocks) * 128, w.n) - 1, p_0 = q.kv - q.n;
    const int j_first = u_first < w.sinks ? u_first : w.lo + u_first - w.sinks, j_last = u_last < w.sinks ? u_last : w.lo + u_last - w.sinks;
    int row_a = max(0, -p_0), row_b = q.n;
    if (a.causal) row_a = max(row_a, j_first - p_0);
    if (a.window > 0 && j_first >= a.sinks)   // (rows from j + window on do not see j)
        row_b = static_cast<int>(min(static_cast<long long>(row_b), static_cast<long long>(j_last) + a.window - p_0));
    c0 = row_a * a.group / 128 * 128;
    tiles = u_last < u_first ? 0 : max(0, (row_b * a.group - c0 + 127) / 128);
}

// The list of blocks, (sequence, head, block), is shared out by what they cost, their tiles of columns: a CTA takes
// the blocks that start in its share of the sum. Every block costs one at least.
struct WeighCost {
    int blocks, even, tiles;    // blocks of a head; the first `even` of them cost `tiles` each (without a window)
    long long head;             // cost of a head
};
__device__ __forceinline__ int weigh_block_cost(const PagedAttnArgs& a, const PagedSeq& q, const PagedSpan& w, int b)
{
    int c0, tiles;
    weigh_columns(a, q, w, b, 1, c0, tiles);
    return max(1, tiles);
}
__device__ __forceinline__ WeighCost weigh_cost(const PagedAttnArgs& a, const PagedSeq& q, const PagedSpan& w)
{
    WeighCost o;
    o.blocks = split_tiles<128>(w.n);
    o.tiles = weigh_block_cost(a, q, w, 0);
    if (a.window > 0)   // (blocks are taken to cost the same)
    {
        o.even = o.blocks;
        o.tiles = 1;
    }
    else o.even = a.causal ? min(o.blocks, max(q.kv - q.n, 0) / 128 + 1) : o.blocks;
    o.head = static_cast<long long>(o.even) * o.tiles;
    for (int b = o.even; b < o.blocks; ++b) o.head += weigh_block_cost(a, q, w, b);
    return o;
}
struct WeighStart {
    long long left;        // the CTA's share not yet taken, in cost, from the block on
    int seq, head, block;
    bool any;
};
// By all of the CTA's threads; scan: shared memory for a long long per warp and two more.
template <int THREADS>
__device__ __forceinline__ WeighStart weigh_start(const PagedAttnArgs& a, long long* scan)
{
    constexpr int WARPS = THREADS / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __shared__ int s_seq;
    auto cost = [&](int s) -> long long {
        PagedSeq q;
        if (s >= a.b.num_seqs || !paged_seq(a.b, s, a.c.page_size, a.c.status, q) || q.n == 0) return 0;
        return weigh_cost(a, q, paged_span(a, q, 0, kWeighAll)).head * a.c.kv_heads;
    };
    const int rounds = (a.b.num_seqs + THREADS - 1) / THREADS;
    long long mine = 0, total = 0;
    for (int r = 0; r < rounds; ++r)
    {
        mine = cost(r * THREADS + tid);
        total += mine;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    if (lane == 0) scan[warp] = total;
    __syncthreads();
    total = 0;
    for (int w = 0; w < WARPS; ++w) total += scan[w];
    const long long x0 = total * blockIdx.x / gridDim.x, x1 = total * (blockIdx.x + 1) / gridDim.x;
    WeighStart o{x1 - x0, 0, 0, 0, x0 < x1};
    if (!o.any) return o;
    long long base = 0;
    for (int r = 0; r < rounds; ++r)
    {
        if (rounds > 1) mine = cost(r * THREADS + tid);
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
        if (x0 >= lo && x0 < lo + mine)
        {
            s_seq = r * THREADS + tid;
            scan[WARPS] = x0 - lo;
        }
        if (x0 < base) break;   // uniform: found in this round
    }
    __syncthreads();
    o.seq = s_seq;
    long long in = scan[WARPS];
    // The first block that starts at x0 or later.
    PagedSeq q;
    o.any = paged_seq(a.b, o.seq, a.c.page_size, nullptr, q) && q.n > 0;   // (else the arrays changed under the call)
    if (!o.any) return o;
    const PagedSpan w = paged_span(a, q, 0, kWeighAll);
    const WeighCost c = weigh_cost(a, q, w);
    o.head = static_cast<int>(in / c.head);
    in -= o.head * c.head;
    o.block = static_cast<int>(min(static_cast<long long>(c.even), (in + c.tiles - 1) / c.tiles));
    long long at = static_cast<long long>(o.block) * c.tiles;
    for (; at < in && o.block < c.blocks; ++o.block) at += weigh_block_cost(a, q, w, o.block);
    o.left -= at - in;
    return o;   // (the block may be the one behind the head's last)
}

template <typename CT, int D>
__global__ void __launch_bounds__(kWeighChunkThreads, 1) paged_weigh_chunk_kernel(const PagedWeighArgs w, const __grid_constant__ WeighTma tma)
{
    using E = WeighChunk<CT, D>;
    constexpr bool CODES = kCodes<CT>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* const smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    const uint32_t sm = smem_u32(smem);
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + E::BAR_OFF);
    uint64_t* const k_full = bars;          // an item's keys and description are there (4 warps)
    uint64_t* const k_empty = bars + 1;     // its products are done
    uint64_t* const d_read = bars + 2;      // its description was read (16 warps)
    uint64_t* const q_full = bars + 4;      // [4] a tile of q and its columns' numbers are there (a warp; by TMA also the bytes)
    uint64_t* const q_empty = bars + 8;     // [4] its products are done
    uint64_t* const s_full = bars + 12;     // [2 tiles][2 blocks] scores are there (the products, and their thread)
    uint64_t* const s_empty = bars + 16;    // [2 tiles][2 blocks] they were read (4 warps)
    uint64_t* const part_full = bars + 20;  // [2 items][2 blocks] sums of the odd tiles are there (4 warps)
    uint64_t* const done = bars + 24;
    uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(bars + 25);
    WeighItem* const items = reinterpret_cast<WeighItem*>(smem + E::ITEM_OFF);
    __shared__ long long scan[kWeighChunkWarps + 1];
    static_assert(sizeof(WeighItem) == 64, "description");
    const PagedAttnArgs& a = w.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (warp == kWeighMmaWarp)
    {
        tmem_alloc(s_tmem, 512);
        tmem_relinquish();
    }
    if (tid == 0)
    {
        mbar_init(k_full, 4);
        mbar_init(k_empty, 1);
        mbar_init(d_read, 16);
        for (int i = 0; i < 4; ++i)
        {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], 1);
            mbar_init(&s_full[i], 2);
            mbar_init(&s_empty[i], 4);
            mbar_init(&part_full[i], 4);
        }
        mbar_init(done, 1);
        fence_mbar_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    pdl_wait();
    pdl_launch();
    const WeighStart st = weigh_start<kWeighChunkThreads>(a, scan);

    if (warp >= kWeighLoadWarp && warp < kWeighMmaWarp)
    {
        // ---------------- loads ----------------
        const int lw = warp - kWeighLoadWarp;
        SplitItem it;
        it.seq = st.seq;
        it.tile = 0;
        it.head = st.head;
        bool more = st.any && paged_seq(a.b, it.seq, a.c.page_size, nullptr, it.q);
        long long left = st.left;
        int block = st.block, price = 1;   // price: of an even block
        // The head's (at its end the next one's) next block, if it is this CTA's.
        auto open = [&] {
            it.w = paged_span(a, it.q, 0, kWeighAll);
            it.tiles = split_tiles<128>(it.w.n);
            price = a.window > 0 ? 1 : 0;
        };
        auto settle = [&] {
            more = more && left > 0;
            if (!more || block < it.tiles) return;
            block = 0;
            if (++it.head == a.c.kv_heads)
            {
                it.head = 0;
                do
                {
                    ++it.seq;
                } while (it.seq < a.b.num_seqs && (!paged_seq(a.b, it.seq, a.c.page_size, nullptr, it.q) || it.q.n == 0));
                more = it.seq < a.b.num_seqs;
                if (more) open();
            }
        };
        if (more)
        {
            open();
            settle();
        }
        bool ok = true;
        int tile_no = 0;   // tiles of earlier items
        int fetched = 0;   // tiles that this warp has sent for
        const bool leader = elect_one();
        for (int item = 0;; ++item)
        {
            WeighItem d{};
            if (more && ok)
            {
                it.cols = it.q.n * a.group;
                d.seq = it.seq; d.head = it.head; d.row0 = it.q.row0; d.kv = it.q.kv; d.n = it.q.n;
                d.keys = it.w.n; d.sinks = it.w.sinks; d.lo = it.w.lo;
                d.block = block;
                // The next block too, if it starts within the share.
                const int cost = price ? price : weigh_block_cost(a, it.q, it.w, block);
                left -= cost;
                d.blocks = 1;
                if (block + 1 < it.tiles && left > 0)
                {
                    d.blocks = 2;
                    left -= price ? price : weigh_block_cost(a, it.q, it.w, block + 1);
                }
                weigh_columns(a, it.q, it.w, block, d.blocks, d.c0, d.tiles);
            }
            // ---- a quarter of the keys: their places, then the copies, when the last item's products are done and every
            // role knows of it (else k_full could run ahead of them) ----
            const int kb = lw >> 1;   // the warp's block, of which it takes 64 keys
            long long off[2] = {-1, -1};
            if (kb < d.blocks)
            {
                const int* const table = a.b.table + it.seq * a.b.table_stride;
#pragma unroll
                for (int y = 0; y < 2; ++y)
                {
                    const int u = (block + kb) * 128 + (lw & 1) * 64 + y * 32 + lane;
                    if (u >= it.w.n) continue;
                    const int j = split_key(it, u), x = a.page_shift >= 0 ? j >> a.page_shift : j / a.c.page_size;
                    const int pg = __ldg(table + x), row = j - x * a.c.page_size;
                    if (pg >= 0 && pg < a.c.num_pages) off[y] = pg * a.c.page_stride + row * a.c.row_stride + it.head * a.c.head_stride;
                    else paged_status(a.c.status, kPagedBadPage);
                }
                __syncwarp();
            }
            if (item > 0) ok = ok && warp_wait(k_empty, (item - 1) & 1, a.c.status) && warp_wait(d_read, (item - 1) & 1, a.c.status);
            if (!ok) d.blocks = 0;
            if (lw == 0 && lane == 0) *items = d;
            if (d.blocks == 0)
            {
                warp_arrive(k_full);
                break;
            }
            if (kb < d.blocks)
            {
                const uint32_t kdst = E::K_OFF + kb * E::BLOCK_B;
#pragma unroll 1
                for (int y = 0; y < 2; ++y)
                {
                    const int r0 = (lw & 1) * 64 + y * 32;
                    constexpr int CPR = D * static_cast<int>(sizeof(CT)) / 16;   // 16-byte pieces of a row in memory
#pragma unroll 4
                    for (int x = 0; x < CPR; ++x)
                    {
                        const int idx = x * 32 + lane, r = idx / CPR, c = idx % CPR;
                        const long long o = __shfl_sync(0xffffffffu, y ? off[1] : off[0], r);
                        const CT* const src = static_cast<const CT*>(a.c.k) + (o < 0 ? 0 : o) + c * (16 / static_cast<int>(sizeof(CT)));
                        if constexpr (!CODES) cp_async16_zfill(sm + kdst + sw128_at(r0 + r, c), src, o >= 0);
                        else
                        {
                            uint4 z = make_uint4(0, 0, 0, 0);
                            if (o >= 0) z = __ldg(reinterpret_cast<const uint4*>(src));
                            auto put = [&](uint32_t lo, uint32_t hi, int piece) {
                                float f[8];
                                decode4<CT>(lo, f);
                                decode4<CT>(hi, f + 4);
                                *reinterpret_cast<uint4*>(smem + kdst + sw128_at(r0 + r, piece)) =
                                    make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
                            };
                            put(z.x, z.y, 2 * c);
                            put(z.z, z.w, 2 * c + 1);
                        }
                    }
                }
                if constexpr (!CODES)
                {
                    cp_commit();
                    cp_wait<0>();
                }
                fence_async_smem();
            }
            warp_arrive(k_full);

            // ---- this warp's tiles of q ----
            for (int x = (lw - tile_no) & 3; x < d.tiles && ok; x += 4)
            {
                const int no = tile_no + x;
                if (no >= 4) ok = warp_wait(&q_empty[lw], (no / 4 - 1) & 1, a.c.status);
                if (!ok) break;
                const int c0 = d.c0 + x * 128;
                float* const info = reinterpret_cast<float*>(smem + E::INFO_OFF + (no & 7) * E::INFO_B);
                const uint32_t qdst = E::Q_OFF + lw * E::BLOCK_B;
                if (tma.on)
                {
                    if (leader)
                    {
                        mbar_expect_tx(&q_full[lw], E::BLOCK_B);
                        const int y = it.head * a.group, z = it.q.row0 + paged_row_of(a, c0);
                        tma_load_3d(sm + qdst, &tma.q, 0, y, z, &q_full[lw]);
                        if constexpr (D == 128) tma_load_3d(sm + qdst + 16384, &tma.q, 64, y, z, &q_full[lw]);
                    }
                    __syncwarp();
                }
                else
                {
                    // Columns lane / QP, + 32 / QP, ...: their rows and heads are counted on.
                    constexpr int QP = E::RB / 16, S = 32 / QP;   // 16-byte pieces of a row
                    int c = lane / QP, row = paged_row_of(a, c0 + c), hg = c0 + c - row * a.group;
                    const __nv_bfloat16* const base = static_cast<const __nv_bfloat16*>(a.q) + it.q.row0 * a.q_row_stride +
                                                      it.head * a.group * a.q_head_stride + lane % QP * 8;
#pragma unroll 4
                    for (int y = 0; y < 128 / S; ++y, c += S)
                    {
                        const bool there = c0 + c < it.cols;
                        cp_async16_zfill(sm + qdst + sw128_at(c, lane % QP), base + (there ? row * a.q_row_stride + hg * a.q_head_stride : 0), there);
                        hg += S;
                        while (hg >= a.group)
                        {
                            hg -= a.group;
                            ++row;
                        }
                    }
                    cp_commit();
                }
                float lse[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) lse[y] = weigh_lse(a, it, min(c0 + lane + 32 * y, it.cols - 1));
#pragma unroll
                for (int y = 0; y < 4; ++y)
                {
                    info[lane + 32 * y] = -lse[y];
                    reinterpret_cast<int*>(info)[128 + lane + 32 * y] = weigh_pos(a, it, c0 + lane + 32 * y);
                }
                if (!tma.on)
                {
                    cp_wait<0>();
                    fence_async_smem();
                }
                warp_arrive(&q_full[lw]);
                ++fetched;
            }
            tile_no += d.tiles;

            block += d.blocks;
            settle();
        }
        cp_wait<0>();
        if (!ok && tma.on && fetched > 0)
            // After a wait that gave up: the block does not end before this warp's copies have landed (or a wait has given up again).
            warp_wait(&q_full[lw], (fetched - 1) & 1, a.c.status);
    }
    else if (warp == kWeighMmaWarp)
    {
        // ---------------- products ----------------
        constexpr uint32_t ID = idesc_f16(true, false, 128, 128);
        const bool leader = elect_one();
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        bool ok = true;
        int no = 0;
        for (int item = 0; ok; ++item)
        {
            ok = warp_wait_spin(k_full, item & 1, a.c.status);
            if (!ok) break;
            const int blocks = __shfl_sync(0xffffffffu, items->blocks, 0), tiles = __shfl_sync(0xffffffffu, items->tiles, 0);
            if (blocks == 0) break;
            for (int x = 0; x < tiles && ok; ++x, ++no)
            {
                const int slot = no & 1, q_slot = no & 3;
                ok = warp_wait_spin(&q_full[q_slot], (no / 4) & 1, a.c.status);
                for (int i = 0; i < 2 && ok; ++i)   // (block 1's scores, where there is none, are passed on unread)
                {
                    if (no >= 2) ok = warp_wait_spin(&s_empty[slot * 2 + i], (no / 2 - 1) & 1, a.c.status);
                    if (!ok) break;
                    tc_fence_after();
                    if (leader)
                    {
                        if (i < blocks)
                        {
                            const uint64_t kd = sw128_desc(sm + E::K_OFF + i * E::BLOCK_B, 16, 1024);
                            const uint64_t qd = sw128_desc(sm + E::Q_OFF + q_slot * E::BLOCK_B, 16, 1024);
#pragma unroll
                            for (int ks = 0; ks < D / 16; ++ks)
                            {
                                const uint64_t o = ((ks >> 2) * 16384 + (ks & 3) * 32) >> 4;
                                umma_f16_ss(tm + (slot * 2 + i) * 128, kd + o, qd + o, ID, ks ? 1u : 0u);
                            }
                        }
                        mbar_arrive(&s_full[slot * 2 + i]);   // (hands on what the loads wrote for the columns)
                        umma_commit(&s_full[slot * 2 + i]);
                    }
                    __syncwarp();
                }
                if (ok && leader) umma_commit(&q_empty[q_slot]);
                __syncwarp();
            }
            if (ok && leader) umma_commit(k_empty);
            __syncwarp();
        }
        if (leader) umma_commit(done);   // nothing is in flight when the tensor memory is freed
        __syncwarp();
        warp_wait_spin(done, 0, a.c.status);
    }
    else
    {
        // ---------------- exponentials and sums of block i, a thread for every other tile of a key ----------------
        const int i = (warp >> 2) & 1, odd = warp >> 3, key = tid & 127;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        bool ok = true;
        int no = 0;
        for (int item = 0; ok; ++item)
        {
            ok = warp_wait(k_full, item & 1, a.c.status);
            if (!ok) break;
            const WeighItem it = *items;
            warp_arrive(d_read);
            if (it.blocks == 0) break;
            // This thread's key: its place, what it has.
            const int u = (it.block + i) * 128 + key;
            const int j = u < it.sinks ? u : it.lo + u - it.sinks, p_0 = it.kv - it.n;
            bool live = false;
            float* at = nullptr;
            float old = 0.f, kf = 1.f, sum = 0.f;
            if (i < it.blocks && u < it.keys)
            {
                const int x = a.page_shift >= 0 ? j >> a.page_shift : j / a.c.page_size, row = j - x * a.c.page_size;
                const int pg = __ldg(a.b.table + it.seq * a.b.table_stride + x);
                live = pg >= 0 && pg < a.c.num_pages;
                if (live && (CODES || !odd))
                {
                    at = w.weights + pg * w.w_page_stride + row * w.w_row_stride + it.head * w.w_head_stride;
                    if (!odd && j < p_0) old = *at;
                    if constexpr (CODES) kf = __ldg(a.c.k_scale + pg * a.c.s_page_stride + row * a.c.s_row_stride + it.head * a.c.s_head_stride);
                }
            }
            // Rows that see the key stand at see_lo .. see_lo + see_n (columns that are not there at -1).
            const unsigned see_lo = a.causal ? j : 0, see_n = a.window > 0 && j >= a.sinks ? a.window - 1 : INT_MAX - see_lo;
            // Tiles [whole_a, whole_b) of the item whose columns are all there and see every key of the block: their rows
            // stand at its last key or later and (window) at most window - 1 behind its first.
            int whole_a = 0, whole_b = 0;
            if (i < it.blocks && (it.block + i + 1) * 128 <= it.keys)
            {
                const int u0 = (it.block + i) * 128, u1 = u0 + 127;
                const int j_first = u0 < it.sinks ? u0 : it.lo + u0 - it.sinks, j_last = u1 < it.sinks ? u1 : it.lo + u1 - it.sinks;
                const int row_a = max(0, (a.causal ? j_last : 0) - p_0);
                const long long row_b = a.window > 0 && j_last >= a.sinks ? static_cast<long long>(j_first) + a.window - p_0 : it.n;
                whole_a = max(0, (row_a * a.group - it.c0 + 127) / 128);
                whole_b = static_cast<int>((max(0ll, min(row_b, static_cast<long long>(it.n))) * a.group - it.c0) / 128);
            }
            for (int x = (no + odd) & 1; x < it.tiles; x += 2)
            {
                const int tile = no + x;
                ok = warp_wait(&s_full[odd * 2 + i], (tile / 2) & 1, a.c.status);
                if (!ok) break;
                tc_fence_after();
                if (i < it.blocks)
                {
                    const uint32_t ts = tmem + (odd * 2 + i) * 128 + lanes;
                    const float* const info = reinterpret_cast<const float*>(smem + E::INFO_OFF + (tile & 7) * E::INFO_B);
                    const bool whole = x >= whole_a && x < whole_b;
                    uint64_t total = 0;   // (a pair of zeros)
                    // In a loop that the instruction caches hold (straight code for all columns waited for instructions).
                    auto columns = [&](auto masked) {
                        const uint64_t log2e = f2(kLog2e, kLog2e), kf2 = f2(kf, kf), scale2 = f2(w.scale, w.scale);
                        auto add = [&](const uint32_t (&r)[32], int q) {
#pragma unroll
                            for (int e = 0; e < 32; e += 4)
                            {
                                const float4 neg = *reinterpret_cast<const float4*>(info + q + e);   // -lse
                                float p[4];
#pragma unroll
                                for (int y = 0; y < 4; y += 2)
                                {
                                    uint64_t z = f2(__uint_as_float(r[e + y]), __uint_as_float(r[e + y + 1]));
                                    if constexpr (CODES) z = f2_mul(z, kf2);
                                    z = f2_fma(z, scale2, y ? f2(neg.z, neg.w) : f2(neg.x, neg.y));
                                    f2_get(f2_mul(z, log2e), p[y], p[y + 1]);
                                    p[y] = ex2(p[y]);
                                    p[y + 1] = ex2(p[y + 1]);
                                }
                                if constexpr (decltype(masked)::value)
                                {
                                    const int4 pos = *reinterpret_cast<const int4*>(reinterpret_cast<const int*>(info) + 128 + q + e);
                                    if (static_cast<unsigned>(pos.x) - see_lo > see_n) p[0] = 0.f;
                                    if (static_cast<unsigned>(pos.y) - see_lo > see_n) p[1] = 0.f;
                                    if (static_cast<unsigned>(pos.z) - see_lo > see_n) p[2] = 0.f;
                                    if (static_cast<unsigned>(pos.w) - see_lo > see_n) p[3] = 0.f;
                                }
                                total = f2_add(total, f2_add(f2(p[0], p[1]), f2(p[2], p[3])));
                            }
                        };
#pragma unroll 1
                        for (int q = 0; q < 128; q += 32)
                        {
                            uint32_t r[32];
                            tmem_ld32(ts + q, r);
                            tmem_ld32_wait(r);
                            add(r, q);
                        }
                    };
                    if (whole) columns(std::false_type{});
                    else columns(std::true_type{});
                    float t0, t1;
                    f2_get(total, t0, t1);
                    sum += t0 + t1;
                    tc_fence_before();
                }
                warp_arrive(&s_empty[odd * 2 + i]);
            }
            no += it.tiles;
            // ---- the two sums of a key ----
            float* const part = reinterpret_cast<float*>(smem + E::PART_OFF) + ((item & 1) * 2 + i) * 128 + key;
            uint64_t* const there = &part_full[(item & 1) * 2 + i];
            if (odd)
            {
                *part = sum;
                warp_arrive(there);
            }
            else
            {
                ok = ok && warp_wait(there, (item / 2) & 1, a.c.status);
                if (live && ok) *at = old + (sum + *part);
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == kWeighMmaWarp)
    {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace hy
