// The k largest entries of each row of a dense matrix as a CSR matrix, columns ascending, and the log of the sum of the row's
// exp(x / temperature).  Equal entries: the lower column; NaN is above all numbers; -0 equals 0.
//
// An entry is compared as 64 bits: its value in an order-preserving code, then the complement of its column, so no two are
// equal and the k largest are always the same k.
// A CTA streams its row, or its part of it, once.  The first 1024 groups of 16 bytes have a largest entry each, and of those comes a bound
// that k entries reach, so few entries of the rest pass it; they are candidates, in shared memory.  A histogram of their keys
// raises the bound (stream_free), or, when they become many, the k largest are kept and the k-th is the new bound (stream_stepwise).
//
// Bound: 4096 x 131072 bf16, k = 64, with the log of the sum: 279 us, 3.85 TB/s, 164 by the bytes: instructions, 52 k a row of which 16 k are the
// exponentials' sums.  777 x 50021 f16, k = 200, without: 53 us, 12 by the bytes: the choice among the candidates, with which each of 1.75
// waves of CTAs ends (three on an SM).  One row of 131072 f32 in a cluster of eight: 14 us.  A step with a barrier each, bounds by selection: 362 us
// for the first.
#include <atomic>

#include "logits.cuh"
#include "rows.cuh"

namespace cb200 {

static __device__ unsigned g_counters[1024];

unsigned *next_counter()
{
    static std::atomic<unsigned> turn{0};
    static std::atomic<unsigned *> base[64];
    int d = 0;
    if (cudaGetDevice(&d) != cudaSuccess || d < 0 || d >= 64) {
        fail("no usable CUDA device (cudaGetDevice failed); libcomet_b200 has no CPU path");
        return nullptr;
    }
    unsigned *p = base[d].load();
    if (!p) {
        const cudaError_t e = cudaGetSymbolAddress((void **)&p, g_counters);
        if (e != cudaSuccess) {
            fail("no usable CUDA device (%s); libcomet_b200 has no CPU path", cudaGetErrorString(e));
            return nullptr;
        }
        base[d] = p;
    }
    return p + turn++ % 1024;
}

static const int MOST_K = 1024, ROOM = 2048;

typedef unsigned long long u64;

// A value in a code whose order as a whole number is the values' order: NaN on top, -0 the same as 0.  Never 0.
template <typename T>
struct Order;
template <>
struct Order<float> {
    static constexpr int BITS = 32, DIGIT = 16;    // DIGIT: 256 digits of the histogram cover a factor of four or so of the value
    static __device__ __forceinline__ uint32_t key(float v)
    {
        const uint32_t u = __float_as_uint(v + 0.0f);
        return v != v ? 0xffffffffu : u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
    }
    static __device__ __forceinline__ float code(uint32_t k) { return value(k); }
    static __device__ __forceinline__ float value(uint32_t k)
    {
        return __uint_as_float(k == 0xffffffffu ? 0x7fffffffu : k ^ ((int32_t)k < 0 ? 0x80000000u : 0xffffffffu));
    }
};
template <typename T, int D>
struct Order16 {
    static constexpr int BITS = 16, DIGIT = D;
    static __device__ __forceinline__ uint32_t key(T v)
    {
        const uint32_t u = *(const uint16_t *)&v;
        if (__hisnan(v)) return 0xffffu;
        return u == 0x8000u ? 0x8000u : u ^ (u & 0x8000u ? 0xffffu : 0x8000u);
    }
    // two at a time
    template <typename T2>
    static __device__ __forceinline__ uint32_t keys(uint32_t u)
    {
        const T2 v = *(const T2 *)&u, zero = {from_float<T>(0.0f), from_float<T>(0.0f)};
        const T2 same = __hadd2(v, zero);          // -0 is 0
        const uint32_t w = *(const uint32_t *)&same, minus = ((w & 0x80008000u) >> 15) * 0xffffu;
        return (w ^ (minus | 0x80008000u)) | __hneu2_mask(v, v);
    }
    static __device__ __forceinline__ T code(uint32_t k)
    {
        const uint16_t u = (uint16_t)(k == 0xffffu ? 0x7fffu : k ^ (k & 0x8000u ? 0x8000u : 0xffffu));
        return *(const T *)&u;
    }
    static __device__ __forceinline__ float value(uint32_t k) { return to_float(code(k)); }
};
template <>
struct Order<__nv_bfloat16> : Order16<__nv_bfloat16, 0> {
    static __device__ __forceinline__ uint32_t keys2(uint32_t u) { return keys<__nv_bfloat162>(u); }
};
template <>
struct Order<__half> : Order16<__half, 3> {
    static __device__ __forceinline__ uint32_t keys2(uint32_t u) { return keys<__half2>(u); }
};

struct TopShared {
    u64 cand[ROOM];
    int hist[256];
    int digit, left, exact;
    int count;
    uint32_t base, bound;          // keys that k entries reach: the first, and the best so far
    float room[3 * TW], m, s, e;
    u64 ends[2 * TW];
    uint32_t least[TW];
};

// Of 256 counts: the highest digit from which on there are at least `want`, how many are above it, and its own; by one warp, in one lane.
__device__ __forceinline__ bool highest_digit(const volatile int *hist, int want, int &digit, int &above, int &own)
{
    const int lane = threadIdx.x & 31;
    int each[8], sum = 0;                          // lane l: the eight digits from 255 - 8 l down
#pragma unroll
    for (int i = 0; i < 8; i++) sum += each[i] = hist[255 - 8 * lane - i];
    int before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    before -= sum;
    if (before >= want || want > before + sum) return false;
    bool done = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if (!done && want <= before + each[i]) {
            done = true;
            digit = 255 - 8 * lane - i;
            above = before;
            own = each[i];
        }
        before += each[i];
    }
    return true;
}

// The least number that exactly k of cand[0..n) reach; 0 if n <= k.  The digits of 8 bits begin where the entries begin to differ
// (they lie between a bound and the largest, so their first bits are alike), and end where a digit tells the k from the rest.
__device__ u64 kth_largest(TopShared &sh, int n, int k)
{
    if (n <= k) return 0;
    const int tid = threadIdx.x;
    u64 lo = ~0ull, hi = 0;
    for (int i = tid; i < n; i += TT) {
        lo = min(lo, sh.cand[i]);
        hi = max(hi, sh.cand[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        lo = min(lo, (u64)__shfl_xor_sync(0xffffffffu, lo, o));
        hi = max(hi, (u64)__shfl_xor_sync(0xffffffffu, hi, o));
    }
    if ((tid & 31) == 0) {
        sh.ends[tid >> 5] = lo;
        sh.ends[TW + (tid >> 5)] = hi;
    }
    sh.hist[tid] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TW; i++) {
        lo = min(lo, sh.ends[i]);
        hi = max(hi, sh.ends[TW + i]);
    }
    int shift = max(0, 56 - __clzll((long long)(hi - lo))), width = 8, left = k;
    u64 found = 0;                                 // (entry - lo) >> (shift + width) of the k-th
    for (;;) {
        for (int i = tid; i < n; i += TT) {
            const u64 v = (sh.cand[i] - lo) >> shift;
            if (v >> width == found) atomicAdd(&sh.hist[(int)v & ((1 << width) - 1)], 1);
        }
        __syncthreads();
        if (tid < 32) {
            int digit, above, own;
            if (highest_digit(sh.hist, left, digit, above, own)) {
                sh.digit = digit;
                sh.left = left - above;
                sh.exact = left - above == own;
            }
        }
        __syncthreads();
        found = found << width | (u64)sh.digit;
        left = sh.left;
        if (sh.exact || shift == 0) return lo + (found << shift);
        width = min(8, shift);
        shift -= width;
        sh.hist[tid] = 0;
        __syncthreads();
    }
}

// The k largest of cand[0..n) to the front, in any order, and count = min(n, k); returns the least number that only they reach.
__device__ u64 keep_largest(TopShared &sh, int n, int k)
{
    const int tid = threadIdx.x;
    if (n <= k) {
        __syncthreads();
        return 0;
    }
    const u64 least = kth_largest(sh, n, k);
    u64 mine[ROOM / TT];
#pragma unroll
    for (int i = 0; i < ROOM / TT; i++) mine[i] = tid + i * TT < n ? sh.cand[tid + i * TT] : 0;
    __syncthreads();
    if (tid == 0) sh.count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROOM / TT; i++)
        if (mine[i] && mine[i] >= least) sh.cand[atomicAdd(&sh.count, 1)] = mine[i];
    __syncthreads();
    return least;
}

// What is summed beside the choice: nothing, exp(x / temperature) (LSE), or all that log probabilities take.
enum { NOTHING, LSE_ONLY, PROBS, PROBS_ENTROPY };
template <int SUM>
struct SumOf {
    typedef ProbSum<SUM == PROBS_ENTROPY> Type;
};
template <>
struct SumOf<NOTHING> {
    typedef LogSum Type;
};
template <>
struct SumOf<LSE_ONLY> {
    typedef LogSum Type;
};

// The first step's bound, by all threads: each of eight warps finds the ceil(k / 8)-th largest of its 128 granules' largest entries, and k
// entries reach the least of those keys.  Of fewer than 256 granules the first warps have 32 each, and only those are asked.
template <typename T>
__device__ __forceinline__ uint32_t first_bound(TopShared &sh, const typename Granule<T>::Most (&gm)[TU], int k, int granules)
{
    const int asked = granules < 32 ? TW : min(TW, granules / 32), want = (k + asked - 1) / asked;
    uint32_t key = 0, gk[TU];
#pragma unroll
    for (int u = 0; u < TU; u++) gk[u] = Order<T>::key(largest(gm[u]));
    for (int bit = Order<T>::BITS - 1; bit >= 0; bit--) {
        const uint32_t more = key | 1u << bit;
        int n = 0;
#pragma unroll
        for (int u = 0; u < TU; u++) n += __popc(__ballot_sync(0xffffffffu, gk[u] >= more));
        if (n >= want) key = more;
        if (n == want) break;
    }
    if ((threadIdx.x & 31) == 0) sh.least[threadIdx.x >> 5] = (int)threadIdx.x >> 5 < asked ? key : 0xffffffffu;
    __syncthreads();
    key = sh.least[0];
#pragma unroll
    for (int i = 1; i < TW; i++) key = min(key, sh.least[i]);
    return key;
}

// Candidates without barriers.  Each one is counted in a histogram of keys above the first bound, and every 64th makes its warp
// look for the highest digit that k entries reach: the other warps' bound from their next step on.  It only rises, and holds
// whenever it is read.  count > ROOM afterwards: the row is one (in order, or of few values) that has to be taken step by step.
template <typename T, int SUM>
__device__ __forceinline__ void stream_free(TopShared &sh, Way<T> &way, int k, int colbits, float c, typename SumOf<SUM>::Type &sum)
{
    constexpr int N = Granule<T>::N, DIGIT = Order<T>::DIGIT;
    const u64 low = (1ull << colbits) - 1;
    volatile uint32_t *bound = &sh.bound;
    const int steps = way.steps();
    uint32_t base = 0;
    bool over = false;
    way.start();
    for (int step = 0; step < steps; step++) {
        const Granule<T> *mine = way.stage(step);
        Granule<T> g[TU];
        typename Granule<T>::Most gm[TU];
#pragma unroll
        for (int u = 0; u < TU; u++) {
            g[u] = mine[u * TT];
            gm[u] = g[u].most();
        }
        if (step == 0) {
            base = first_bound<T>(sh, gm, k, way.end - way.begin);
            if (threadIdx.x == 0) sh.base = *bound = base;
            __syncthreads();
        }
        if (SUM) sum.add(g, most_of(most_of(gm[0], gm[1]), most_of(gm[2], gm[3])), c);
        if (over) continue;
        const T least = Order<T>::code(*bound);
        unsigned pending = 0;
#pragma unroll
        for (int u = 0; u < TU; u++)
            if (reaches(gm[u], least)) pending |= g[u].at_least(least) << (u * N);
        if (!__any_sync(0xffffffffu, pending != 0)) continue;
        bool look = false;
        while (pending) {
            const int b = __ffs(pending) - 1, u = b / N, e = b % N, col = way.column(step, u, e);
            pending &= pending - 1;
            if (col < 0 || col >= way.ncols) continue;
            const uint32_t key = Order<T>::key(((const T *)&mine[u * TT])[e]);
            if (key < base) continue;              // nothing is smaller than a bound that is NaN
            const int at = atomicAdd(&sh.count, 1);
            if (at < ROOM) sh.cand[at] = (u64)key << colbits | (low - (unsigned)col);
            atomicAdd(&sh.hist[min((key - base) >> DIGIT, 255u)], 1);
            look |= at % 64 == 63;
        }
        if (__any_sync(0xffffffffu, look)) {
            int digit, above, own;
            if (highest_digit(sh.hist, k, digit, above, own)) atomicMax((unsigned *)bound, base + ((uint32_t)digit << DIGIT));
            __syncwarp();
            over = __any_sync(0xffffffffu, *(volatile int *)&sh.count > ROOM);         // the same in every lane
            if (!SUM && over) break;
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
}

// Candidates step by step: when they become many, the k largest are kept and the k-th of them is the new bound.  Holds for
// every row and k.  Leaves the k largest.
template <typename T, int SUM>
__device__ __noinline__ void stream_stepwise(TopShared &sh, Way<T> &way, int k, int colbits, float c, typename SumOf<SUM>::Type &sum)
{
    constexpr int N = Granule<T>::N;
    const u64 low = (1ull << colbits) - 1;
    const int steps = way.steps(), limit = min(max(2 * k, 256), ROOM);
    u64 bound = 0;                                 // an entry has to be larger
    T least_value = Order<T>::code(0xffffffffu);   // the bound's value; NaN: all are larger
    if (threadIdx.x == 0) sh.count = 0;
    way.start();
    for (int step = 0; step < steps; step++) {
        const Granule<T> *mine = way.stage(step);
        Granule<T> g[TU];
        typename Granule<T>::Most gm[TU];
#pragma unroll
        for (int u = 0; u < TU; u++) {
            g[u] = mine[u * TT];
            gm[u] = g[u].most();
        }
        if (step == 0) {
            const uint32_t key = first_bound<T>(sh, gm, k, way.end - way.begin);
            bound = (u64)key << colbits;
            least_value = Order<T>::code(key);
        }
        if (SUM) sum.add(g, most_of(most_of(gm[0], gm[1]), most_of(gm[2], gm[3])), c);
        unsigned pending = 0;
#pragma unroll
        for (int u = 0; u < TU; u++) pending |= g[u].at_least(least_value) << (u * N);
        for (;;) {
            bool full = false;
            unsigned without = 0;                  // entries that found no room
            while (pending) {
                const int b = __ffs(pending) - 1, u = b / N, e = b % N, col = way.column(step, u, e);
                pending &= pending - 1;
                const u64 it = (u64)Order<T>::key(((const T *)&mine[u * TT])[e]) << colbits | (low - (unsigned)col);
                if (it > bound && col >= 0 && col < way.ncols) {
                    const int at = atomicAdd(&sh.count, 1);
                    full |= at >= limit - 1;
                    if (at < ROOM) sh.cand[at] = it;
                    else without |= 1u << b;
                }
            }
            if (!__syncthreads_or(full)) break;
            const u64 least = keep_largest(sh, min(sh.count, ROOM), k);
            if (least > bound + 1) {
                bound = least - 1;
                least_value = Order<T>::code((uint32_t)(bound >> colbits));
            }
            pending = without;
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    keep_largest(sh, sh.count, k);
}

// Long rows, or many entries of them: a CTA, or a cluster of them, per row.
template <typename T, int SUM, bool FREE>
__global__ void __launch_bounds__(TT, 3)
top_kernel(int64_t nrows, int ncols, int slice, const T *__restrict__ xs, int64_t ldx, int k, int colbits, float c, float inv, int64_t *__restrict__ pos,
           int64_t *__restrict__ crd, float *__restrict__ val, float *__restrict__ lse, const ProbCall probs)
{
    constexpr bool PROB = SUM >= PROBS;
    extern __shared__ __align__(128) uint4 ring[];  // a warp reads 512 bytes at a time: from a line on, or a fifth line takes an eighth more time
    __shared__ TopShared sh;
    const int tid = threadIdx.x;
    const unsigned rank = cluster_rank(), ranks = cluster_size();
    const int64_t t = blockIdx.x / ranks;
    const T *x = xs + t * ldx;
    Way<T> way;
    way.ring = ring;
    way.from = (const uint4 *)((uintptr_t)x & ~(uintptr_t)15);
    way.off = (int)((uintptr_t)x & 15) / (int)sizeof(T);
    way.ncols = ncols;
    way.all = (way.off + ncols + Way<T>::N - 1) / Way<T>::N;
    way.begin = min((int)rank * slice, way.all);
    way.end = min(way.begin + slice, way.all);
    typename SumOf<SUM>::Type sum;
    if constexpr (PROB) sum.start();
    else sum = {MINUS_INF, 0.0f, make_float2(0.0f, 0.0f)};
    const u64 low = (1ull << colbits) - 1;
    if (FREE) {
        sh.hist[tid] = 0;
        if (tid == 0) {
            sh.count = 0;
            sh.base = sh.bound = 0;
        }
        __syncthreads();
        stream_free<T, SUM>(sh, way, k, colbits, c, sum);
        const int n = sh.count;
        __syncthreads();                           // all have read it
        if (n > ROOM) {
            LogSum none;
            stream_stepwise<T, NOTHING>(sh, way, k, colbits, c, none);
        } else if (n > k) {                        // those that do not reach the last bound go
            if (tid < 32) {
                int digit, above, own;
                if (highest_digit(sh.hist, k, digit, above, own)) sh.bound = sh.base + ((uint32_t)digit << Order<T>::DIGIT);
            }
            u64 mine[ROOM / TT];
#pragma unroll
            for (int i = 0; i < ROOM / TT; i++) mine[i] = tid + i * TT < n ? sh.cand[tid + i * TT] : 0;
            __syncthreads();
            const u64 least = (u64)sh.bound << colbits;
            if (tid == 0) sh.count = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < ROOM / TT; i++)
                if (mine[i] > least) sh.cand[atomicAdd(&sh.count, 1)] = mine[i];
            __syncthreads();
            if (sh.count > ROOM / MOST_CLUSTER) keep_largest(sh, sh.count, k);
        }
    } else {
        stream_stepwise<T, SUM>(sh, way, k, colbits, c, sum);
    }
    float m = sum.m, s = 0.0f, ent = 0.0f;
    if constexpr (PROB) sum.total(s, ent);
    else s = sum.s.x + sum.s.y;
    if (PROB) {
        float r[1] = {m}, q[2];
        cta_reduce<1, TW, true>(r, sh.room);
        shift_to(r[0], m, c, s, ent);
        q[0] = s;
        q[1] = ent;
        cta_reduce<2, TW, false>(q, sh.room + TW);
        m = r[0];
        s = q[0];
        ent = q[1];
        if (tid == 0) {
            sh.m = m;
            sh.s = s;
            sh.e = ent;
        }
    } else if (SUM) {
        float r[1] = {m}, q[1];
        cta_reduce<1, TW, true>(r, sh.room);
        q[0] = m == MINUS_INF ? 0.0f : s * exp2_fast((m - r[0]) * c);
        cta_reduce<1, TW, false>(q, sh.room + TW);
        m = r[0];
        s = q[0];
        if (tid == 0) {
            sh.m = m;
            sh.s = s;
        }
    }
    if (ranks > 1) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (rank == 0) {
            // what the others have, all at once: lane r of each warp asks CTA r, and warp r copies its candidates
            static_assert(TW >= MOST_CLUSTER, "a warp for each CTA");
            const int lane = tid & 31, from = tid >> 5;
            const bool other = lane > 0 && lane < (int)ranks;
            const int theirs = other ? peer_load(&sh.count, lane) : 0, have = sh.count;
            float om = MINUS_INF, os = 0.0f, oe = 0.0f;
            if (SUM && other) {
                om = peer_load(&sh.m, lane);
                os = peer_load(&sh.s, lane);
                if (PROB) oe = peer_load(&sh.e, lane);
            }
            int upto = theirs;
#pragma unroll
            for (int o = 1; o < MOST_CLUSTER; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const int all = have + __shfl_sync(0xffffffffu, upto, MOST_CLUSTER - 1);
            if (all <= ROOM) {
                const int n = __shfl_sync(0xffffffffu, theirs, from), at = have + __shfl_sync(0xffffffffu, upto, from) - n;
                for (int i = lane; i < n; i += 32) sh.cand[at + i] = peer_load(&sh.cand[i], from);
                __syncthreads();
                if (tid == 0) sh.count = all;
                __syncthreads();
            } else {
                const int most = max(k, ROOM / MOST_CLUSTER);    // candidates of a CTA
                for (unsigned r = 1; r < ranks; r++) {
                    const int n = peer_load(&sh.count, r), have = sh.count;
                    for (int i = tid; i < n; i += TT) sh.cand[have + i] = peer_load(&sh.cand[i], r);
                    __syncthreads();
                    if (tid == 0) sh.count = have + n;
                    __syncthreads();
                    if (sh.count > ROOM - most) keep_largest(sh, sh.count, k);
                }
            }
            for (unsigned r = 1; SUM && r < ranks; r++) {
                const float rm = __shfl_sync(0xffffffffu, om, r), nm = max_nan(m, rm);
                float rs = __shfl_sync(0xffffffffu, os, r), re = __shfl_sync(0xffffffffu, oe, r);
                if (PROB) {
                    shift_to(nm, m, c, s, ent);
                    shift_to(nm, rm, c, rs, re);
                    s += rs;
                    ent += re;
                } else {
                    s = (m == MINUS_INF ? 0.0f : s * exp2_fast((m - nm) * c)) + (rm == MINUS_INF ? 0.0f : rs * exp2_fast((rm - nm) * c));
                }
                m = nm;
            }
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (rank != 0) return;
    }
    if (SUM == LSE_ONLY && tid == 0) lse[t] = log_of_sum(m, s, inv);
    const RowProb p(m, s, ent);
    if (PROB) give_probs(probs, t, x, ncols, p, inv, tid, TT);
    auto value = [&](uint32_t key) { return PROB ? p.of(Order<T>::value(key), inv) : Order<T>::value(key); };
    if (tid == 0) {
        pos[t] = t * k;
        if (t == nrows - 1) pos[nrows] = nrows * k;
    }
    int n = sh.count;
    if (n > TT && n > k) {
        keep_largest(sh, n, k);
        n = k;
    }
    // by column, ascending: the complement of the column, descending
    if (n <= TT) {
        u64 it = tid < n ? sh.cand[tid] : 0;
        if (n > k) {                               // those with fewer than k above them, to that place
            int above = 0;
            if ((tid & ~31) < n)
                for (int i = 0; i < n; i++) above += sh.cand[i] > it;
            __syncthreads();
            if (it && above < k) sh.cand[above] = it;
            __syncthreads();
            it = tid < k ? sh.cand[tid] : 0;
        }
        if (it) {
            int at = 0;
            for (int i = 0; i < min(n, k); i++) at += (sh.cand[i] & low) > (it & low);
            crd[t * k + at] = (int64_t)(low - (it & low));
            val[t * k + at] = value((uint32_t)(it >> colbits));
        }
        return;
    }
    int room = 1;
    while (room < k) room *= 2;
    u64 *v = sh.cand + MOST_K;
    for (int i = tid; i < room; i += TT) {
        const u64 it = i < k ? sh.cand[i] : 0;
        v[i] = i < k ? (low - (it & low)) << 32 | it >> colbits : ~0ull;
    }
    __syncthreads();
    for (int size = 2; size <= room; size *= 2)
        for (int step = size / 2; step > 0; step /= 2) {
            for (int i = tid; i < room / 2; i += TT) {
                const int lo = i / step * step * 2 + i % step, hi = lo + step;
                const u64 a = v[lo], b = v[hi];
                if ((a > b) == ((lo & size) == 0)) {
                    v[lo] = b;
                    v[hi] = a;
                }
            }
            __syncthreads();
        }
    for (int i = tid; i < k; i += TT) {
        crd[t * k + i] = (int64_t)(v[i] >> 32);
        val[t * k + i] = value((uint32_t)v[i]);
    }
}

// An entry of a short row, larger ones first, of equal values the lower column: 16-bit values and the column in one word, which is never 0;
// others in two, of which only the first is compared where the columns are in order already.
template <typename T>
struct Short {
    uint32_t word;
    __device__ __forceinline__ void set(T v, int col) { word = Order<T>::key(v) << 16 | (0xffffu - col); }
    __device__ __forceinline__ void none() { word = 0; }
    __device__ __forceinline__ uint32_t most() const { return word; }
    __device__ __forceinline__ int column(uint32_t) const { return 0; }
    static __device__ __forceinline__ void order(Short &a, Short &b)
    {
        const uint32_t x = max(a.word, b.word);
        b.word = min(a.word, b.word);
        a.word = x;
    }
};
template <>
struct Short<float> {
    uint32_t word;
    int col;
    __device__ __forceinline__ void set(float v, int c)
    {
        word = Order<float>::key(v);
        col = c;
    }
    __device__ __forceinline__ void none() { word = 0; }
    __device__ __forceinline__ uint32_t most() const { return word; }
    static __device__ __forceinline__ void order(Short &a, Short &b)
    {
        if (b.word > a.word || (b.word == a.word && b.col < a.col)) {
            const Short x = a;
            a = b;
            b = x;
        }
    }
};

// Short rows and few entries of them (a router's choices): a warp per row, R consecutive columns a lane, so that of equal entries
// the lowest lane's is the lowest column's.  Each lane sorts its own (odd-even merges), and k times the warp takes the largest of its
// lanes' first ones.
//
// Bound: instructions; 65536 rows of 256 and k = 8 in bf16 take 27 us, 6 by the bytes; 65 when the lane that gives an entry looked for its next
// one.  16384 rows of 64 in f32: 10 us on the device.
template <typename T, int R, int SUM>
__global__ void __launch_bounds__(128)
top_short_kernel(int64_t nrows, int ncols, const T *__restrict__ xs, int64_t ldx, bool whole, int k, float c, float inv, int64_t *__restrict__ pos,
                 int64_t *__restrict__ crd, float *__restrict__ val, float *__restrict__ lse, const ProbCall probs)
{
    constexpr bool ONE = Order<T>::BITS == 16;
    const int lane = threadIdx.x & 31;
    const int64_t t = ((int64_t)blockIdx.x * 128 + threadIdx.x) >> 5;
    if (t >= nrows) return;
    const T *x = xs + t * ldx;
    struct alignas(sizeof(T) * R < 16 ? sizeof(T) * R : 16) Part {
        T v[R];
    } part;
    if (whole && lane * R + R <= ncols) {
        part = ((const Part *)x)[lane];
    } else {
#pragma unroll
        for (int r = 0; r < R; r++) part.v[r] = lane * R + r < ncols ? x[lane * R + r] : from_float<T>(MINUS_INF);
    }
    Short<T> own[R];
    if constexpr (ONE && R > 1) {
#pragma unroll
        for (int r = 0; r < R; r += 2) {
            const uint32_t keys = Order<T>::keys2(((const uint32_t *)&part)[r / 2]), col = lane * R + r;
            own[r].word = keys << 16 | (0xffffu - col);
            own[r + 1].word = (keys & 0xffff0000u) | (0xfffeu - col);
        }
    } else {
#pragma unroll
        for (int r = 0; r < R; r++) own[r].set(part.v[r], lane * R + r);
    }
    if (lane * R + R > ncols)
#pragma unroll
        for (int r = 0; r < R; r++)
            if (lane * R + r >= ncols) own[r].none();
#pragma unroll
    for (int p = 1; p < R; p *= 2)
#pragma unroll
        for (int q = p; q > 0; q /= 2)
#pragma unroll
            for (int j = q % p; j + q < R; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; i++)
                    if (i + j + q < R && (i + j) / (2 * p) == (i + j + q) / (2 * p)) Short<T>::order(own[i + j], own[i + j + q]);
    int col = 0;
    uint32_t got = 0;                              // lane i: the i-th largest
    for (int i = 0; i < k; i++) {
        const uint32_t top = __reduce_max_sync(0xffffffffu, own[0].most());
        bool mine = own[0].most() == top;
        int at = 0;
        if constexpr (!ONE) {
            const int who = __ffs(__ballot_sync(0xffffffffu, mine)) - 1;
            at = __shfl_sync(0xffffffffu, own[0].col, who);
            mine = lane == who;
        }
        if (lane == i) {
            col = ONE ? (int)(0xffffu - (top & 0xffffu)) : at;
            got = ONE ? top >> 16 : top;
        }
        if (mine) {
#pragma unroll
            for (int r = 0; r + 1 < R; r++) own[r] = own[r + 1];
            own[R - 1].none();
        }
    }
    RowProb p(MINUS_INF, 0.0f, 0.0f);
    if (SUM) {
        float m = MINUS_INF, s = 0.0f, ent = 0.0f;
#pragma unroll
        for (int r = 0; r < R; r++) m = max_nan(m, to_float(part.v[r]));
        m = warp_max(m);
        if (SUM == LSE_ONLY) {
#pragma unroll
            for (int r = 0; r < R; r++) s += exp2_fast((to_float(part.v[r]) - m) * c);
            s = warp_sum(s);
            if (lane == 0) lse[t] = log_of_sum(m, s, inv);
        } else {
#pragma unroll
            for (int r = 0; r < R; r++) {
                const float d = (to_float(part.v[r]) - m) * c, q = exp2_fast(d);
                s += q;
                if (SUM == PROBS_ENTROPY) ent = fmaf(q, fmaxf(d, -16384.0f), ent);
            }
            s = warp_sum(s);
            if (SUM == PROBS_ENTROPY) ent = warp_sum(ent);
            p = RowProb(m, s, ent);
            give_probs(probs, t, x, ncols, p, inv, lane, 32);
        }
    }
    int place = 0;
    for (int i = 0; i < k; i++) place += __shfl_sync(0xffffffffu, col, i) < col;
    if (lane < k) {
        crd[t * k + place] = col;
        val[t * k + place] = SUM >= PROBS ? p.of(Order<T>::value(got), inv) : Order<T>::value(got);
    }
    if (lane == 0) {
        pos[t] = t * k;
        if (t == nrows - 1) pos[nrows] = nrows * k;
    }
}

struct TopCall {
    int64_t nrows;
    int ncols;
    const void *x;
    int64_t ldx;
    int k;
    float c, inv;
    int64_t *pos, *crd;
    float *val, *lse;
    cudaStream_t st;
    int sum;
    ProbCall probs;
};

template <typename T, int R>
static void launch_short(const TopCall &a)
{
    const size_t piece = sizeof(T) * R < 16 ? sizeof(T) * R : 16;
    const bool whole = (uintptr_t)a.x % piece == 0 && a.ldx * (int64_t)sizeof(T) % (int64_t)piece == 0;
    const unsigned grid = (unsigned)ceil_div(a.nrows, 4);
    auto kernel = a.sum == NOTHING ? top_short_kernel<T, R, NOTHING> : a.sum == LSE_ONLY ? top_short_kernel<T, R, LSE_ONLY> : a.sum == PROBS ? top_short_kernel<T, R, PROBS>
                                                                                                                              : top_short_kernel<T, R, PROBS_ENTROPY>;
    kernel<<<grid, 128, 0, a.st>>>(a.nrows, a.ncols, (const T *)a.x, a.ldx, whole, a.k, a.c, a.inv, a.pos, a.crd, a.val, a.lse, a.probs);
}

template <typename T, int SUM>
static int launch_long(const TopCall &a)
{
    constexpr int N = Granule<T>::N;
    const int all = (a.ncols + 2 * N - 2) / N;     // granules of a row, wherever it starts
    int ranks = 1, colbits = 1;
    while (ranks < MOST_CLUSTER && a.nrows * ranks <= sm_count() && all / ranks >= 2 * TU * TT) ranks *= 2;
    while ((1 << colbits) <= a.ncols) colbits++;
    const size_t smem = (size_t)STAGES * TU * TT * 16;
    if (a.nrows * ranks > 0x7fffffffLL) return fail("top_entries: more than 2^31 rows");
    // beyond 256 entries the candidates of a row without barriers would not fit their room
    auto kernel = a.k <= 256 ? top_kernel<T, SUM, true> : top_kernel<T, SUM, false>;
    return launch_cluster(kernel, (unsigned)(a.nrows * ranks), ranks, TT, smem, smem, a.st, a.nrows, a.ncols, (int)ceil_div(all, ranks),
                          (const T *)a.x, a.ldx, a.k, colbits, a.c, a.inv, a.pos, a.crd, a.val, a.lse, a.probs);
}

template <typename T>
static int launch_top(const TopCall &a)
{
    // By warps / by CTAs, 4096 rows, k = 8 and 32, us: 512 columns of bf16 5.7, 9.7 / 128, 131, 1024 of bf16 24, 34 / 137, 143 (the CTAs' bound was looser);
    // 512 of f32 -, 24 / -, 124, 1024 of f32 93, 148 / 49, 58: a warp's two words an entry fill its registers.
    if (a.ncols > (sizeof(T) == 2 ? 1024 : 512) || a.k > 32)
        return a.sum == NOTHING ? launch_long<T, NOTHING>(a) : a.sum == LSE_ONLY ? launch_long<T, LSE_ONLY>(a) : a.sum == PROBS ? launch_long<T, PROBS>(a)
                                                                                                              : launch_long<T, PROBS_ENTROPY>(a);
    if (a.ncols <= 32) launch_short<T, 1>(a);
    else if (a.ncols <= 64) launch_short<T, 2>(a);
    else if (a.ncols <= 128) launch_short<T, 4>(a);
    else if (a.ncols <= 256) launch_short<T, 8>(a);
    else if (a.ncols <= 512) launch_short<T, 16>(a);
    else if constexpr (sizeof(T) == 2) launch_short<T, 32>(a);
    CB_LAUNCH_CHECK();
    return 0;
}

// log_probs with alternatives: the choice and the sums in one pass
template <typename T>
int top_log_probs(int64_t nrows, int ncols, const T *x, int64_t ldx, int k, float c, float inv, int64_t *pos, int64_t *crd, float *val, const ProbCall &probs,
                  cudaStream_t st)
{
    return launch_top<T>({nrows, ncols, x, ldx, k, c, inv, pos, crd, val, nullptr, st, probs.entropy ? PROBS_ENTROPY : PROBS, probs});
}
template int top_log_probs(int64_t, int, const __nv_bfloat16 *, int64_t, int, float, float, int64_t *, int64_t *, float *, const ProbCall &, cudaStream_t);
template int top_log_probs(int64_t, int, const __half *, int64_t, int, float, float, int64_t *, int64_t *, float *, const ProbCall &, cudaStream_t);
template int top_log_probs(int64_t, int, const float *, int64_t, int, float, float, int64_t *, int64_t *, float *, const ProbCall &, cudaStream_t);

template <typename T>
static int top_entries(int64_t nrows, int64_t ncols, const void *x, int64_t ldx, int64_t k, const double *temperature, int64_t *pos, int64_t *crd,
                       float *val, float *lse, void *stream)
{
    clear_error();
    cudaStream_t st = (cudaStream_t)stream;
    if (nrows < 0 || ncols <= 0 || ncols >= 1LL << 30) return fail("top_entries: %lld rows of %lld columns", (long long)nrows, (long long)ncols);
    if (ldx < ncols) return fail("top_entries: leading dimension smaller than the number of columns");
    if (k < 1 || k > ncols || k > MOST_K) return fail("top_entries: %lld entries a row; 1 to %d, and no more than a row has", (long long)k, MOST_K);
    if (nrows > 0x7fffffffLL) return fail("top_entries: more than 2^31 rows");
    if (lse && !temperature) return fail("top_entries: the sum needs a temperature");
    if (temperature && !temperature_fits(*temperature)) return fail("top_entries: temperature %g is not a number of 1e-38 to 1e30", *temperature);
    if ((uintptr_t)x % sizeof(T)) return fail("top_entries: an address that is not a multiple of the element's size");
    if (nrows == 0) {
        CB_CUDA(cudaMemsetAsync(pos, 0, sizeof(int64_t), st));
        return 0;
    }
    TopCall a = {nrows, (int)ncols, x, ldx, (int)k, 0.0f, 0.0f, pos, crd, val, lse, st, lse ? LSE_ONLY : NOTHING, {}};
    if (lse) {
        a.c = (float)(LOG2E_D / *temperature);
        a.inv = (float)(1.0 / *temperature);
    }
    return launch_top<T>(a);
}

}  // namespace cb200

#define TOP(suffix, T)                                                                                                                  \
    extern "C" int32_t comet_b200_dev_top_entries_##suffix##_i64(int64_t nrows, int64_t ncols, const void *x, int64_t ldx, int64_t k,    \
                                                                 const double *temperature, int64_t *pos, int64_t *crd, float *val,      \
                                                                 float *lse, void *stream)                                               \
    {                                                                                                                                    \
        return cb200::top_entries<T>(nrows, ncols, x, ldx, k, temperature, pos, crd, val, lse, stream);                                  \
    }
TOP(bf16, __nv_bfloat16)
TOP(f16, __half)
TOP(f32, float)
