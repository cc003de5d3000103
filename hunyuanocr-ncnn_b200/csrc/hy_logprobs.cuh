// Log probabilities of given tokens, entropy and top alternatives of rows of logits.
//
// With M a row's largest logit, c the count of logits equal to it, and over the
// others s = sum e^(x - M) and t = sum (M - x) e^(x - M):
//   log prob of x = (x - M) - log(c + s),   entropy = log(c + s) + t / (c + s).
// s and t hold no term of the largest logit, so that what is left beside a probability
// near 1 keeps its relative precision (log(1 + s) is taken as log1p), and no large terms
// cancel. One pass: every thread keeps (c, s, t) of its own elements against the largest m that
// its warp has met, rescaled when that grows; they are joined at the end. (With a largest of
// its own for every thread some lane has a new one in nearly every step, and the whole warp pays for it.)
//
// The alternatives come from the same pass: what is stored of every group of 128
// elements is its maximum (in shared memory). The n-th largest of the threads' maxima
// is a lower bound of the row's n-th largest element, so the groups whose maximum
// reaches it - hardly more than n - hold all that is looked for, and only they are read
// again, a vector to a thread. A list that overflows (thousands of equal logits) is left aside for n
// passes that take one element each.
//
// A row belongs to a cluster of 1 to 8 CTAs, which meet in the shared memory of the first. Memory bounds it where
// there are many rows: 1024 of 120818 fp32 logits take 75 us without alternatives, 6.6 TB/s, 81 with 8; bf16 56 and 62:
// half the bytes but as many exponentials (their units are busy half of the time) and 62% of the issue slots, a warp waiting
// mostly for its loads, of which the registers (60) let eight CTAs be under way. One row with 20 alternatives: 9 us, one latency after another.
#pragma once

#include <cooperative_groups.h>

#include "hy_paged.cuh"

namespace hy {

constexpr int kLogprobManyThreads = 128;   // of a CTA, eight to an SM: while some are in their last steps, others load
constexpr int kLogprobFewThreads = 512;    // where there are fewer CTAs than SMs: a row's loads are all on their way at once
constexpr int kLogprobRun = 4;         // steps of a group: 128 elements
constexpr int kLogprobGroups = 256;    // groups that are read again by all threads together
constexpr int kLogprobList = 512;      // candidates of a CTA
constexpr int kLogprobMaxTop = 64;
constexpr int kLogprobMaxCluster = 8;

struct LogprobArgs {
    const void* logits;
    long long row_stride;
    int rows, vocab;
    const int* tokens;
    int tokens_per_row, top;
    float* logprobs;
    float* entropy;
    int* top_ids;
    float* top_logprobs;
    int split;   // CTAs of a row
    int iters;   // steps of a CTA (groups of a thread)
};

// Largest of three, two; a NaN among them comes out.
__device__ __forceinline__ float max_nan(float a, float b, float c)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Largest of a warp's; a NaN among them comes out.
__device__ __forceinline__ float warp_max_nan(float x)
{
    float r;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Order of the alternatives: by value, then the lower index (zeros of both signs are equal). 0: none.
__device__ __forceinline__ unsigned long long logprob_key(float x, int index)
{
    const uint32_t b = __float_as_uint(x + 0.f);
    return (static_cast<unsigned long long>(b & 0x80000000u ? ~b : b | 0x80000000u) << 32) | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ float logprob_key_value(unsigned long long k)
{
    const uint32_t b = static_cast<uint32_t>(k >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

// What a set of logits amounts to (see above).
struct LogprobState {
    float m, c, s, t;
};
__device__ __forceinline__ void logprob_raise(LogprobState& o, float m)   // m > o.m
{
    // (where f is 0 the way from o.m to m may be infinite)
    const float f = exp2_approx((o.m - m) * 1.4426950408889634f), all = o.s + o.c;
    o.t = f > 0.f ? f * (o.t + (m - o.m) * all) : 0.f;
    o.s = f * all;
    o.c = 0.f;
    o.m = m;
}

// A row of logits as 16-byte vectors from the aligned address at or before its start.
template <typename T>
struct LogprobRow {
    static constexpr int EV = 16 / static_cast<int>(sizeof(T));
    static constexpr uint32_t NONE = EV == 4 ? 0xff800000u : 0xff80ff80u;   // a word of -infinity
    const T* base;   // aligned
    int skip, end;   // elements of the row: [skip, end) from base

    __device__ __forceinline__ LogprobRow(const T* row, int vocab)
    {
        skip = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
        base = row - skip;
        end = skip + vocab;
    }
    __device__ __forceinline__ int vectors() const { return (end + EV - 1) / EV; }
    // Vector v as fp32; -infinity outside the row.
    __device__ __forceinline__ uint4 raw(int v) const
    {
        if (v * EV >= skip && (v + 1) * EV <= end) return __ldg(reinterpret_cast<const uint4*>(base + v * EV));
        uint32_t w[4] = {NONE, NONE, NONE, NONE};
#pragma unroll
        for (int e = 0; e < EV; ++e)
        {
            const int x = v * EV + e;
            if (x < skip || x >= end) continue;
            if constexpr (EV == 4) w[e] = __float_as_uint(__ldg(reinterpret_cast<const float*>(base) + x));
            else
            {
                const uint32_t b = __ldg(reinterpret_cast<const unsigned short*>(base) + x);
                w[e >> 1] = (e & 1) ? (w[e >> 1] & 0xffffu) | (b << 16) : (w[e >> 1] & 0xffff0000u) | b;
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ void unpack(const uint4& x, float* f)
    {
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < EV; ++e)
            f[e] = EV == 4 ? __uint_as_float(w[e]) : __uint_as_float((e & 1) ? w[e >> 1] & 0xFFFF0000u : w[e >> 1] << 16);
    }
};

// Block-wide maximum (a NaN comes out); red: shared memory of a float per warp.
template <int kLogprobThreads>
__device__ __forceinline__ float logprob_block_max(float x, float* red)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = max_nan(x, __shfl_xor_sync(0xffffffffu, x, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
    __syncthreads();
    x = red[0];
#pragma unroll
    for (int w = 1; w < kLogprobThreads / 32; ++w) x = max_nan(x, red[w]);
    __syncthreads();
    return x;
}

template <typename T, bool TOP, int kLogprobThreads>
__global__ void __launch_bounds__(kLogprobThreads, 1024 / kLogprobThreads) logprob_kernel(const LogprobArgs a)
{
    namespace cg = cooperative_groups;
    using Row = LogprobRow<T>;
    constexpr int EV = Row::EV, U = 32 / EV, NW = kLogprobThreads / 32;
    extern __shared__ __align__(16) float group_max[];   // [groups of a thread][threads]
    __shared__ float red[3 * NW];
    __shared__ __align__(16) float thread_max[kLogprobThreads];
    __shared__ LogprobState parts[kLogprobMaxCluster];             // (the first CTA's are used)
    __shared__ unsigned long long list[TOP ? kLogprobList : 1];    // candidates
    __shared__ __align__(16) unsigned long long tops[TOP ? kLogprobMaxCluster * kLogprobMaxTop : 1];   // (the first CTA's) sorted lists
    __shared__ unsigned long long mine[TOP ? kLogprobMaxTop : 1], best[NW];
    __shared__ int group_list[TOP ? kLogprobGroups : 1];           // groups that may hold some of the top
    __shared__ int count, groups;
    __shared__ float bound;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = blockIdx.x % a.split, r = blockIdx.x / a.split;
    if (a.split > 1) cg::this_cluster().barrier_arrive();   // (the first CTA runs before the others write to its shared memory)
    pdl_wait();
    const Row row(static_cast<const T*>(a.logits) + r * a.row_stride, a.vocab);
    const int nv = row.vectors(), per = a.iters * kLogprobThreads * U;
    const int v0 = rank * per, v1 = min(nv, v0 + per);   // this CTA's vectors

    LogprobState st = {-INFINITY, 0.f, 0.f, 0.f};
    float own_max = -INFINITY, run_max = -INFINITY;
    // (the first token's logit, ahead of the row's)
    const int token0 = rank == 0 && tid < a.tokens_per_row ? __ldg(a.tokens + static_cast<long long>(r) * a.tokens_per_row + tid) : -1;
    const float logit0 = token0 >= 0 && token0 < a.vocab ? to_f32<T>(static_cast<const T*>(a.logits)[r * a.row_stride + token0]) : 0.f;
    for (int it = 0; it < a.iters; ++it)
    {
        const int v = v0 + it * kLogprobThreads * U + tid;
        uint4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            x[u] = v + u * kLogprobThreads < v1 ? row.raw(v + u * kLogprobThreads) : make_uint4(Row::NONE, Row::NONE, Row::NONE, Row::NONE);
        float f[U * EV];
#pragma unroll
        for (int u = 0; u < U; ++u) Row::unpack(x[u], f + u * EV);
        float m0 = max_nan(f[0], f[1]), m1 = max_nan(f[2], f[3]);
#pragma unroll
        for (int e = 4; e < U * EV; e += 4)
        {
            m0 = max_nan(m0, f[e], f[e + 1]);
            m1 = max_nan(m1, f[e + 2], f[e + 3]);
        }
        const float top = max_nan(m0, m1);
        if constexpr (TOP)
        {
            run_max = max_nan(run_max, top);
            if (it % kLogprobRun == kLogprobRun - 1 || it == a.iters - 1)
            {
                group_max[it / kLogprobRun * kLogprobThreads + tid] = run_max;
                own_max = max_nan(own_max, run_max);
                run_max = -INFINITY;
            }
        }
        const float most = warp_max_nan(top);   // (what follows is alike in the whole warp)
        if (most < st.m)
        {
            // x - m, its exponential, the sums; -1000 stands for less (the exponential is 0: 0 times infinity is not taken).
            const uint64_t neg = f2(-st.m, -st.m), log2e = f2(1.4426950408889634f, 1.4426950408889634f);
            uint64_t s2 = 0, t2 = 0;   // (pairs of zeros)
#pragma unroll
            for (int e = 0; e < U * EV; e += 2)
            {
                float d0, d1, y0, y1;
                f2_get(f2_add(f2(f[e], f[e + 1]), neg), d0, d1);
                d0 = fmaxf(d0, -1000.f);
                d1 = fmaxf(d1, -1000.f);
                const uint64_t d = f2(d0, d1);
                f2_get(f2_mul(d, log2e), y0, y1);
                const uint64_t p = f2(exp2_approx(y0), exp2_approx(y1));
                s2 = f2_add(s2, p);
                t2 = f2_fma(d, p, t2);
            }
            float y0, y1;
            f2_get(s2, y0, y1);
            st.s += y0 + y1;
            f2_get(t2, y0, y1);
            st.t -= y0 + y1;
        }
        else if (most != -INFINITY)   // the first finite ones, a new maximum, one more like it, a NaN
        {
            if (!(most <= st.m) && st.m == st.m) logprob_raise(st, most);   // (a NaN stays one)
            float s = 0.f, t = 0.f;
#pragma unroll
            for (int e = 0; e < U * EV; ++e)
            {
                const float d = fmaxf(f[e] - st.m, -1000.f), p = exp2_approx(d * 1.4426950408889634f);
                const bool same = f[e] == st.m;
                st.c += same ? 1.f : 0.f;
                s += same ? 0.f : p;
                t -= same ? 0.f : d * p;
            }
            st.s += s;
            st.t += t;
        }
    }

    // ---- the CTA's state ----
    if constexpr (TOP)
    {
        if (a.top > kLogprobThreads / 16) thread_max[tid] = own_max;
        else
        {
            float x = max_nan(own_max, __shfl_xor_sync(0xffffffffu, own_max, 1));
            x = max_nan(x, __shfl_xor_sync(0xffffffffu, x, 2));
            if ((tid & 3) == 0) thread_max[tid >> 2] = x;
        }
    }
    const float M = logprob_block_max<kLogprobThreads>(st.m, red);   // (also makes group_max and thread_max visible)
    if (st.m != M) logprob_raise(st, M);
    float sum[3] = {st.c, st.s, st.t};
#pragma unroll
    for (int i = 0; i < 3; ++i)
    {
        sum[i] = warp_sum(sum[i]);
        if (lane == 0) red[i * NW + warp] = sum[i];
    }
    if (tid == 0) count = groups = 0;
    if constexpr (TOP)
    {
        // The n-th largest of the maxima of runs of 4 threads (of single threads where n is large).
        const int many = a.top > kLogprobThreads / 16 ? kLogprobThreads : kLogprobThreads / 4;
        if (tid < many)
        {
            const float own = thread_max[tid];
            int above = 0;
#pragma unroll 4
            for (int j = 0; j < many; j += 4)
            {
                const float4 o = *reinterpret_cast<const float4*>(thread_max + j);
                above += (o.x > own || (o.x == own && j < tid)) + (o.y > own || (o.y == own && j + 1 < tid)) +
                         (o.z > own || (o.z == own && j + 2 < tid)) + (o.w > own || (o.w == own && j + 3 < tid));
            }
            if (above == a.top - 1) bound = own;
        }
    }
    __syncthreads();
    if (a.split > 1) cg::this_cluster().barrier_wait();
    if (tid == 0)
    {
        LogprobState p = {M, 0.f, 0.f, 0.f};
        for (int w = 0; w < NW; ++w)
        {
            p.c += red[w];
            p.s += red[NW + w];
            p.t += red[2 * NW + w];
        }
        *cg::this_cluster().map_shared_rank(&parts[rank], 0) = p;
    }
    if constexpr (TOP)
    {
        // (with a NaN in the row nothing below is used; `bound` may then hold anything)
        const bool usable = M == M && M != -INFINITY && M != INFINITY;
        const float low = usable ? bound : INFINITY;
        const int all_groups = (a.iters + kLogprobRun - 1) / kLogprobRun * kLogprobThreads;
        auto look = [&](int g, int x, auto&& take) {   // vector x of group g
            const int it = g / kLogprobThreads * kLogprobRun + x / U, v = v0 + (it * U + x % U) * kLogprobThreads + g % kLogprobThreads;
            if (it >= a.iters || v >= v1) return;
            float f[EV];
            Row::unpack(row.raw(v), f);
#pragma unroll
            for (int e = 0; e < EV; ++e)
                if (f[e] >= low && f[e] != -INFINITY) take(logprob_key(f[e], v * EV + e - row.skip));
        };
        auto each = [&](auto&& take) {   // every element of this CTA's that may be among the top
            for (int g = tid; g < all_groups; g += kLogprobThreads)
            {
                if (!(group_max[g] >= low) || group_max[g] == -INFINITY) continue;
#pragma unroll 1
                for (int x = 0; x < U * kLogprobRun; ++x) look(g, x, take);
            }
        };
        auto note = [&](unsigned long long key) {
            const int i = atomicAdd(&count, 1);
            if (i < kLogprobList) list[i] = key;
        };
        for (int g = tid; g < all_groups; g += kLogprobThreads)
            if (group_max[g] >= low && group_max[g] != -INFINITY)
            {
                const int i = atomicAdd(&groups, 1);
                if (i < kLogprobGroups) group_list[i] = g;
            }
        __syncthreads();
        if (groups <= kLogprobGroups)
        {
            // A vector of a group to a thread, so that all loads are on their way at once.
#pragma unroll 4
            for (int x = tid; x < groups * U * kLogprobRun; x += kLogprobThreads) look(group_list[x / (U * kLogprobRun)], x % (U * kLogprobRun), note);
        }
        else each(note);
        if (tid < kLogprobMaxTop) mine[tid] = 0;
        __syncthreads();
        const int n = count;
        if (n <= kLogprobList)
        {
            for (int i = tid; i < n; i += kLogprobThreads)
            {
                const unsigned long long key = list[i];
                int above = 0;
                for (int j = 0; j < n; ++j) above += list[j] > key;
                if (above < a.top) mine[above] = key;
            }
            __syncthreads();
        }
        else
        {
            unsigned long long last = ~0ull;
            for (int k = 0; k < a.top; ++k)
            {
                unsigned long long next = 0;
                each([&](unsigned long long key) {
                    if (key < last && key > next) next = key;
                });
#pragma unroll
                for (int o = 16; o > 0; o >>= 1)
                {
                    const unsigned long long other = __shfl_xor_sync(0xffffffffu, next, o);
                    next = other > next ? other : next;
                }
                if (lane == 0) best[warp] = next;
                __syncthreads();
                for (int w = 0; w < NW; ++w) next = best[w] > next ? best[w] : next;
                if (tid == 0) mine[k] = next;
                last = next;
                __syncthreads();
            }
        }
        if (tid < a.top) cg::this_cluster().map_shared_rank(tops, 0)[rank * a.top + tid] = mine[tid];
    }
    if (a.split > 1) cg::this_cluster().sync();
    else __syncthreads();
    if (rank != 0) return;

    // ---- the row's answer, by its first CTA ----
    float top = parts[0].m;
    for (int p = 1; p < a.split; ++p) top = max_nan(top, parts[p].m);
    const bool usable = top == top && top != INFINITY && top != -INFINITY;
    float c = 0.f, s = 0.f, t = 0.f;
    for (int p = 0; p < a.split; ++p)
    {
        LogprobState o = parts[p];
        if (o.m != top) logprob_raise(o, top);
        c += o.c;
        s += o.s;
        t += o.t;
    }
    const float nan = __int_as_float(0x7fffffff);
    const float less = usable ? (c == 1.f ? log1pf(s) : logf(c + s)) : nan;
    if (tid == 0 && a.entropy) a.entropy[r] = usable ? less + t / (c + s) : nan;
    for (int i = tid; i < a.tokens_per_row; i += kLogprobThreads)
    {
        const int token = i == tid ? token0 : __ldg(a.tokens + static_cast<long long>(r) * a.tokens_per_row + i);
        float lp = nan;
        if (usable && token >= 0 && token < a.vocab)
            lp = ((i == tid ? logit0 : to_f32<T>(static_cast<const T*>(a.logits)[r * a.row_stride + token])) - top) - less;
        a.logprobs[static_cast<long long>(r) * a.tokens_per_row + i] = lp;
    }
    if constexpr (TOP)
    {
        auto put = [&](int i, unsigned long long key) {
            const long long at = static_cast<long long>(r) * a.top + i;
            const bool there = usable && key != 0;
            a.top_ids[at] = there ? static_cast<int>(~static_cast<uint32_t>(key)) : -1;
            a.top_logprobs[at] = there ? (logprob_key_value(key) - top) - less : usable ? -INFINITY : nan;
        };
        // The CTAs' sorted lists into one: an entry's place is the number of larger ones.
        const int n = a.split * a.top;
        int total = 0;
        for (int i0 = 0; i0 < n; i0 += kLogprobThreads)
        {
            const int i = i0 + tid;
            const unsigned long long key = i < n ? tops[i] : 0;
            total += __syncthreads_count(key != 0);
            if (key == 0) continue;
            int above = 0, j = 0;
#pragma unroll 4
            for (; j + 2 <= n; j += 2)
            {
                const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(tops + j);
                above += (o.x > key) + (o.y > key);
            }
            if (j < n) above += tops[j] > key;
            if (above < a.top) put(above, key);
        }
        for (int i = (usable ? total : 0) + tid; i < a.top; i += kLogprobThreads) put(i, 0);
    }
}

}  // namespace hy
