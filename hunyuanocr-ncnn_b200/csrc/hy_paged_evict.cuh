// Eviction from the paged cache: of every sequence and KV head the `keep`
// positions that count most stay, and their rows move to the positions 0 .. keep - 1 in the
// order they had.
//
// A cluster of 1 to 8 CTAs takes a (sequence, head). Its first CTA selects: the weights, as
// whole numbers of the same order, lie in registers (the first 8192 of them, the next 24576 in shared memory, more are
// read again each time); the keep-th largest is found bit by bit
// (the count of those that reach a candidate decides each bit, and the search ends as soon as
// a candidate leaves exactly `keep`; two bits at a time gained nothing), and the kept positions are written in order,
// a rank being the number of kept ones before. Among equal weights the lower positions stay.
//
// Then all CTAs of the cluster move rows, each some 16-byte columns of them: a row moves to its own
// place or a lower one, so rows are taken in ascending runs, a run's loads (all of them) before its
// stores; what a later run reads lies behind what an earlier one writes. Rows before the
// first evicted position stay where they are.
//
// One record cut from 4111 to 1024 positions of 8 heads (bf16): some 21 us, look-ups, search, ranks and moves
// one after another; 64 records of 900-1152 (E4M3): 45 us.
#pragma once

#include <cooperative_groups.h>

#include "hy_paged.cuh"

namespace hy {

constexpr int kEvictThreads = 512;
constexpr int kEvictHeld = 16;      // weights that a thread holds in registers
constexpr int kEvictMore = 24 * 1024;   // weights behind those that the CTA holds in shared memory, at most
constexpr int kEvictMaxCluster = 8;
constexpr int kEvictInFlight = 4;   // 16-byte pieces of a thread in a run

struct PagedEvictArgs {
    PagedCache c;
    PagedBatch b;
    float* weights;
    long long w_page_stride, w_head_stride, w_row_stride;
    int* kept;       // [num_seqs][kv_heads][keep]
    int* kv_len;     // written by evict_lengths_kernel
    int keep, first, recent;
    int elem;        // bytes of an element of k and v
    int pieces;      // 16-byte pieces of a row
    int page_shift;  // log2 of page_size, or -1
    int cluster;
    int more;        // weights that shared memory holds
};

// Weights as whole numbers of the same order (zeros of both signs equal, a NaN least).
__device__ __forceinline__ uint32_t evict_order(float w)
{
    if (w != w) return 0;
    const uint32_t b = __float_as_uint(w + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct EvictPlace {
    int page, row;
};

// Sum over the block; red: shared memory of an int per warp, free again on return.
__device__ __forceinline__ int evict_block_sum(int x, int* red)
{
    x = __reduce_add_sync(0xffffffffu, x);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
    __syncthreads();
    int all = __reduce_add_sync(0xffffffffu, (threadIdx.x & 31) < kEvictThreads / 32 ? red[threadIdx.x & 31] : 0);
    __syncthreads();
    return all;
}

__global__ void __launch_bounds__(kEvictThreads, 2) paged_evict_kernel(const PagedEvictArgs a)
{
    namespace cg = cooperative_groups;
    constexpr int T = kEvictThreads, W = T / 32, R = kEvictHeld, CHUNK = T * R;
    extern __shared__ uint32_t more[];
    __shared__ int red[W], counts[R * W];
    __shared__ int changed;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = blockIdx.x % a.cluster, item = blockIdx.x / a.cluster;
    const int seq = item / a.c.kv_heads, head = item - seq * a.c.kv_heads;
    pdl_wait();
    const int kv = __ldg(a.b.kv_len + seq);
    const int* const table = a.b.table + seq * a.b.table_stride;
    int* const kept = a.kept + static_cast<long long>(item) * a.keep;
    auto place = [&](int j) -> EvictPlace {
        const int x = a.page_shift >= 0 ? j >> a.page_shift : j / a.c.page_size;
        return {__ldg(table + x), j - x * a.c.page_size};
    };

    // ---- sequences that have nothing to give, or do not hold (alike in the whole cluster) ----
    bool bad = kv < 0 || kv > static_cast<long long>(a.b.table_width) * a.c.page_size;
    if (bad && tid == 0) paged_status(a.c.status, kPagedBadLength);
    if (!bad && kv > a.keep)
    {
        bool lost = false;
        for (int x = tid; x < (kv + a.c.page_size - 1) / a.c.page_size; x += T)
        {
            const int pg = __ldg(table + x);
            lost |= pg < 0 || pg >= a.c.num_pages;
        }
        bad = __syncthreads_or(lost);
        if (bad && tid == 0) paged_status(a.c.status, kPagedBadPage);
    }
    if (bad || kv <= a.keep)
    {
        if (rank == 0)
            for (int i = tid; i < a.keep; i += T) kept[i] = !bad && i < kv ? i : -1;
        return;
    }

    auto weight_at = [&](EvictPlace p) { return a.weights + p.page * a.w_page_stride + p.row * a.w_row_stride + head * a.w_head_stride; };
    if (rank == 0)
    {
        auto fresh = [&](int j) -> uint32_t {
            return j < a.first || j >= kv - a.recent ? 0xffffffffu : evict_order(*weight_at(place(j)));
        };
#pragma unroll 4
        for (int j = CHUNK + tid; j < min(kv, CHUNK + a.more); j += T) more[j - CHUNK] = fresh(j);   // (for this thread alone)
        auto key = [&](int j) -> uint32_t { return j >= kv ? 0 : j >= CHUNK && j - CHUNK < a.more ? more[j - CHUNK] : fresh(j); };
        // Position i * T + tid of a run of CHUNK; those of the first run are held.
        // (All look-ups, then all weights, so that they are on their way together.)
        uint32_t held[R];
        {
            EvictPlace at[R];
            float wt[R];
#pragma unroll
            for (int i = 0; i < R; ++i) at[i] = i * T < kv ? place(min(i * T + tid, kv - 1)) : EvictPlace{0, 0};
#pragma unroll
            for (int i = 0; i < R; ++i) wt[i] = i * T < kv ? *weight_at(at[i]) : 0.f;
#pragma unroll
            for (int i = 0; i < R; ++i)
            {
                const int j = i * T + tid;
                held[i] = j >= kv ? 0 : j < a.first || j >= kv - a.recent ? 0xffffffffu : evict_order(wt[i]);
            }
        }
        auto reach = [&](uint32_t least) {   // how many keys reach `least` (not 0)
            int n = 0;
#pragma unroll
            for (int i = 0; i < R; ++i) n += held[i] >= least;
            for (int j = CHUNK + tid; j < kv; j += T) n += key(j) >= least;
            return evict_block_sum(n, red);
        };
        uint32_t least = 0;
        int n_least = kv;   // keys that reach it
        for (uint32_t bit = 0x80000000u; bit && n_least != a.keep; bit >>= 1)
        {
            const int n = reach(least | bit);
            if (n >= a.keep)
            {
                least |= bit;
                n_least = n;
            }
        }
        // Of those equal to the least, the lowest positions stay.
        int equal = n_least == a.keep ? kv : a.keep - (least == 0xffffffffu ? 0 : reach(least + 1));
        int done = 0;       // kept positions of earlier runs
        for (int j0 = 0; j0 < kv; j0 += CHUNK)
        {
            uint32_t stays = 0;   // bit i: position j0 + i * T + tid stays
            // Ranks within the run: the flags' bits before this one, warp by warp, i by i.
            auto ranks = [&](uint32_t flags, int (&before)[R]) {
#pragma unroll
                for (int i = 0; i < R; ++i)
                {
                    const uint32_t in = __ballot_sync(0xffffffffu, (flags >> i) & 1u);
                    before[i] = __popc(in & ((1u << lane) - 1u));
                    if (lane == 0) counts[i * W + warp] = __popc(in);
                }
                __syncthreads();
                int all = 0;
                if (warp == 0)
                {
                    for (int x = 0; x < R * W; x += 32)
                    {
                        const int n = counts[x + lane];
                        int inc = n;
#pragma unroll
                        for (int d = 1; d < 32; d <<= 1)
                        {
                            const int v = __shfl_up_sync(0xffffffffu, inc, d);
                            if (lane >= d) inc += v;
                        }
                        counts[x + lane] = all + inc - n;
                        all += __shfl_sync(0xffffffffu, inc, 31);
                    }
                    if (lane == 0) red[0] = all;
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < R; ++i) before[i] += counts[i * W + warp];
                all = red[0];
                __syncthreads();
                return all;
            };
            uint32_t same = 0;
#pragma unroll
            for (int i = 0; i < R; ++i)
            {
                const int j = j0 + i * T + tid;
                const uint32_t k = j0 == 0 ? held[i] : key(j);
                if (j < kv && k > least) stays |= 1u << i;
                if (j < kv && k == least) same |= 1u << i;
            }
            int before[R];
            if (n_least == a.keep) stays |= same;
            else
            {
                const int all = ranks(same, before);
#pragma unroll
                for (int i = 0; i < R; ++i)
                    if (((same >> i) & 1u) && before[i] < equal) stays |= 1u << i;
                equal -= min(equal, all);
            }
            const int all = ranks(stays, before);
#pragma unroll
            for (int i = 0; i < R; ++i)
                if ((stays >> i) & 1u) kept[done + before[i]] = j0 + i * T + tid;
            done += all;
        }
    }
    if (tid == 0) changed = a.keep;
    cg::this_cluster().sync();   // the list is there

    // ---- the first position whose row is another ----
    int start = a.keep;
    for (int i = tid; i < a.keep; i += T)
        if (kept[i] != i)
        {
            start = i;
            break;
        }
    atomicMin(&changed, start);
    __syncthreads();
    start = changed;

    // ---- rows: this CTA's columns of K and V ----
    const int cols = 2 * a.pieces / a.cluster, c0 = rank * cols;   // pieces of K, then of V
    const int per = T / cols * kEvictInFlight;                     // rows of a run
    const int my_row = tid / cols, my_piece = c0 + tid % cols;
    const bool isv = my_piece >= a.pieces, mover = my_row < T / cols;
    unsigned char* const pool = static_cast<unsigned char*>(isv ? a.c.v : a.c.k) + (my_piece - (isv ? a.pieces : 0)) * 16;
    auto row_at = [&](int j) -> uint4* {
        const EvictPlace p = place(j);
        return reinterpret_cast<uint4*>(pool + (p.page * a.c.page_stride + p.row * a.c.row_stride + head * a.c.head_stride) * a.elem);
    };
    for (int i0 = start; i0 < a.keep; i0 += per)
    {
        uint4 x[kEvictInFlight];
#pragma unroll
        for (int u = 0; u < kEvictInFlight; ++u)
        {
            const int i = i0 + u * (T / cols) + my_row;
            if (mover && i < a.keep) x[u] = *row_at(kept[i]);
        }
        __syncthreads();   // the run was read
#pragma unroll
        for (int u = 0; u < kEvictInFlight; ++u)
        {
            const int i = i0 + u * (T / cols) + my_row;
            if (mover && i < a.keep) *row_at(i) = x[u];
        }
    }
    // ---- weights and scales, by the first CTA ----
    if (rank != 0) return;
    for (int i0 = start; i0 < a.keep; i0 += T)
    {
        const int i = i0 + tid;
        float w = 0.f, ks = 0.f, vs = 0.f;
        auto scale_at = [&](EvictPlace p) { return p.page * a.c.s_page_stride + p.row * a.c.s_row_stride + head * a.c.s_head_stride; };
        if (i < a.keep)
        {
            const EvictPlace p = place(kept[i]);
            w = *weight_at(p);
            if (a.c.k_scale)
            {
                ks = a.c.k_scale[scale_at(p)];
                vs = a.c.v_scale[scale_at(p)];
            }
        }
        __syncthreads();
        if (i < a.keep)
        {
            const EvictPlace p = place(i);
            *weight_at(p) = w;
            if (a.c.k_scale)
            {
                a.c.k_scale[scale_at(p)] = ks;
                a.c.v_scale[scale_at(p)] = vs;
            }
        }
    }
}

// Lengths of the sequences that were cut. (Apart: every head's CTAs read the old ones.)
__global__ void evict_lengths_kernel(const PagedEvictArgs a)
{
    pdl_wait();
    const int s = blockIdx.x * blockDim.x + threadIdx.x;
    if (s >= a.b.num_seqs) return;
    const int* const kept = a.kept + static_cast<long long>(s) * a.c.kv_heads * a.keep;
    if (a.kv_len[s] > a.keep && kept[0] >= 0) a.kv_len[s] = a.keep;
}

}  // namespace hy
