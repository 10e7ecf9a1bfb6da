// The k largest entries of each row of a dense matrix as a CSR matrix, columns ascending, and the log of the sum of the row's
// exp(x / temperature).  Equal entries: the lower column; NaN is above all numbers; -0 equals 0.
//
// An entry is compared as 64 bits: its value in an order-preserving code, then the complement of its column, so no two are
// equal and the k largest are always the same k.
// A CTA streams its row, or its part of it, once.  The first 512 groups of 16 bytes have a largest entry each, and of those comes a bound
// that k entries reach, so few entries of the rest pass it; they are candidates, in shared memory.  When they become many, the
// k largest are kept and the k-th of them is the new bound.
#include <atomic>

#include "logits.cuh"

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

static const int TT = 256, TW = TT / 32, TU = 2, STAGES = 4, MOST_K = 1024, ROOM = 2048, MOST_RANKS = 8;

typedef unsigned long long u64;

// A value in a code whose order as a whole number is the values' order: NaN on top, -0 the same as 0.  Never 0.
template <typename T>
struct Order;
template <>
struct Order<float> {
    static constexpr int BITS = 32;
    static __device__ __forceinline__ uint32_t key(float v)
    {
        const uint32_t u = __float_as_uint(v + 0.0f);
        return v != v ? 0xffffffffu : u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
    }
    static __device__ __forceinline__ float value(uint32_t k)
    {
        return __uint_as_float(k == 0xffffffffu ? 0x7fffffffu : k ^ ((int32_t)k < 0 ? 0x80000000u : 0xffffffffu));
    }
};
template <typename T>
struct Order16 {
    static constexpr int BITS = 16;
    static __device__ __forceinline__ uint32_t key(T v)
    {
        const uint32_t u = *(const uint16_t *)&v;
        if (__hisnan(v)) return 0xffffu;
        return u == 0x8000u ? 0x8000u : u ^ (u & 0x8000u ? 0xffffu : 0x8000u);
    }
    static __device__ __forceinline__ float value(uint32_t k)
    {
        const uint16_t u = (uint16_t)(k == 0xffffu ? 0x7fffu : k ^ (k & 0x8000u ? 0x8000u : 0xffffu));
        return to_float(*(const T *)&u);
    }
};
template <>
struct Order<__nv_bfloat16> : Order16<__nv_bfloat16> {};
template <>
struct Order<__half> : Order16<__half> {};

struct TopShared {
    u64 cand[ROOM];
    int hist[256];
    int digit, left, exact;
    int count;
    float room[2 * TW], m, s;
    u64 ends[2 * TW];
    uint32_t least[TW];
};

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
        if (tid < 32) {                            // lane l: the eight digits from 255 - 8 l down
            int own[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) sum += own[i] = sh.hist[255 - 8 * tid - i];
            int before = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, before, o);
                if (tid >= o) before += v;
            }
            before -= sum;
            if (before < left && left <= before + sum) {
                bool done = false;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (!done && left <= before + own[i]) {
                        done = true;
                        sh.digit = 255 - 8 * tid - i;
                        sh.left = left - before;
                        sh.exact = left - before == own[i];
                    }
                    before += own[i];
                }
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
    const u64 least = kth_largest(sh, n, k);
    u64 mine[ROOM / TT];
#pragma unroll
    for (int i = 0; i < ROOM / TT; i++) mine[i] = threadIdx.x + i * TT < n ? sh.cand[threadIdx.x + i * TT] : 0;
    __syncthreads();
    if (n <= k) return 0;
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROOM / TT; i++)
        if (mine[i] && mine[i] >= least) sh.cand[atomicAdd(&sh.count, 1)] = mine[i];
    __syncthreads();
    return least;
}

// Long rows, or many entries of them: a cluster of CTAs per row, each streams a part of it through a ring of stages in shared memory
// (a thread copies 16 bytes and reads the same 16, so the ring needs no barriers).
template <typename T, bool LSE>
__global__ void __launch_bounds__(TT)
top_kernel(int64_t nrows, int ncols, int slice, const T *__restrict__ xs, int64_t ldx, int k, int colbits, float c, float inv, int64_t *__restrict__ pos,
           int64_t *__restrict__ crd, float *__restrict__ val, float *__restrict__ lse)
{
    constexpr int N = Granule<T>::N;
    extern __shared__ uint4 ring[];                // STAGES * TU * TT
    __shared__ TopShared sh;
    const int tid = threadIdx.x;
    const unsigned rank = cluster_rank(), ranks = cluster_size();
    const int64_t t = blockIdx.x / ranks;
    const T *x = xs + t * ldx;
    const int off = (int)((uintptr_t)x & 15) / (int)sizeof(T), all = (off + ncols + N - 1) / N;
    const int begin = min((int)rank * slice, all), end = min(begin + slice, all);
    const uint4 *from = (const uint4 *)((uintptr_t)x & ~(uintptr_t)15);
    const int limit = min(max(4 * k, 512), ROOM);  // more candidates than this are cut to k
    if (tid == 0) sh.count = 0;
    auto fetch = [&](int step) {
#pragma unroll
        for (int u = 0; u < TU; u++) {
            const int i = begin + (step * TU + u) * TT + tid;
            if (i < end) copy_granule(ring + ((step % STAGES) * TU + u) * TT + tid, from + i);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) fetch(i);
    __syncthreads();
    u64 bound = 0;                                 // an entry has to be larger
    uint32_t boundkey = 0;
    float m = MINUS_INF, s = 0.0f;
    const int steps = (end - begin + TU * TT - 1) / (TU * TT);
    for (int step = 0; step < steps; step++) {
        fetch(step + STAGES - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        Granule<T> g[TU];
        uint32_t gk[TU];
#pragma unroll
        for (int u = 0; u < TU; u++) {
            const int i = begin + (step * TU + u) * TT + tid;
            if (i < end) g[u].w = ring[((step % STAGES) * TU + u) * TT + tid];
            if (i == 0 || i >= all - 1 || i >= end) {          // entries before and behind the row
                float v[N];
                g[u].unpack(v);
#pragma unroll
                for (int e = 0; e < N; e++)
                    if (i >= end || i * N + e < off || i * N + e >= off + ncols) v[e] = MINUS_INF;
                g[u].pack(v);
            }
            const T gm = granule_max(g[u]);
            gk[u] = Order<T>::key(gm);
            if (LSE) {
                const float nm = max_nan(m, to_float(gm));
                if (nm != m) {
                    s *= exp2_fast((m - nm) * c);
                    m = nm;
                }
                if (m != MINUS_INF) {
                    float v[N];
                    g[u].unpack(v);
#pragma unroll
                    for (int e = 0; e < N; e++) s += exp2_fast((v[e] - m) * c);
                }
            }
        }
        if (step == 0) {
            // Each warp finds the ceil(k / 8)-th largest of its 64 groups' largest entries; k entries reach the least of those eight.
            const int want = (k + TW - 1) / TW;
            uint32_t key = 0;
            if (want <= 32 * TU)
                for (int bit = Order<T>::BITS - 1; bit >= 0; bit--) {
                    const uint32_t more = key | 1u << bit;
                    int n = 0;
#pragma unroll
                    for (int u = 0; u < TU; u++) n += __popc(__ballot_sync(0xffffffffu, gk[u] >= more));
                    if (n >= want) key = more;
                    if (n == want) break;
                }
            if ((tid & 31) == 0) sh.least[tid >> 5] = key;
            __syncthreads();
            boundkey = sh.least[0];
#pragma unroll
            for (int i = 1; i < TW; i++) boundkey = min(boundkey, sh.least[i]);
            bound = (u64)boundkey << colbits;
        }
        unsigned pending = 0;
        bool full = false;
        auto look = [&](bool put) {
#pragma unroll
            for (int u = 0; u < TU; u++) {
                if (put ? !(pending >> (u * N) & ((1u << N) - 1)) : gk[u] < boundkey) continue;
                const T *v = (const T *)&g[u].w;
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const int col = (begin + (step * TU + u) * TT + tid) * N + e - off;
                    const u64 it = (u64)Order<T>::key(v[e]) << colbits | (u64)((1u << colbits) - 1 - (unsigned)col);
                    const unsigned bit = 1u << (u * N + e);
                    if (!put) {
                        if (it > bound && col >= 0 && col < ncols) pending |= bit;
                    } else if (pending & bit) {
                        const int at = atomicAdd(&sh.count, 1);
                        full |= at >= limit - 1;
                        if (at < ROOM) {
                            sh.cand[at] = it;
                            pending &= ~bit;
                        }
                    }
                }
            }
        };
        look(false);
        for (;;) {
            if (pending) look(true);
            if (!__syncthreads_or(full || pending != 0)) break;
            const u64 least = keep_largest(sh, min(sh.count, ROOM), k);
            if (least > bound + 1) bound = least - 1;
            boundkey = (uint32_t)(bound >> colbits);
            full = false;
            if (pending) {                         // of those that found no room, the ones that are still large enough
                const unsigned without = pending;
                pending = 0;
                look(false);
                pending &= without;
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    keep_largest(sh, sh.count, k);
    if (LSE) {
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
        if (rank == 0)
            for (unsigned r = 1; r < ranks; r++) {             // the others' candidates, as many as fit at a time
                const int n = peer_load(&sh.count, r), have = sh.count;
                for (int i = tid; i < n; i += TT) sh.cand[have + i] = peer_load(&sh.cand[i], r);
                __syncthreads();
                if (tid == 0) sh.count = have + n;
                __syncthreads();
                if (sh.count > ROOM - k || r == ranks - 1) keep_largest(sh, sh.count, k);
                if (LSE) {
                    const float om = peer_load(&sh.m, r), os = peer_load(&sh.s, r), nm = max_nan(m, om);
                    s = (m == MINUS_INF ? 0.0f : s * exp2_fast((m - nm) * c)) + (om == MINUS_INF ? 0.0f : os * exp2_fast((om - nm) * c));
                    m = nm;
                }
            }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (rank != 0) return;
    }
    if (LSE && tid == 0) lse[t] = m == MINUS_INF ? m : fmaf(log2f(s), LN2, m * inv);
    if (tid == 0) {
        pos[t] = t * k;
        if (t == nrows - 1) pos[nrows] = nrows * k;
    }
    // by column, ascending: the complement of the column, descending
    const u64 low = (1ull << colbits) - 1;
    if (k <= TT) {
        u64 it = 0;
        int at = 0;
        if (tid < k) {
            it = sh.cand[tid];
            for (int i = 0; i < k; i++) at += (sh.cand[i] & low) > (it & low);
            crd[t * k + at] = (int64_t)(low - (it & low));
            val[t * k + at] = Order<T>::value((uint32_t)(it >> colbits));
        }
        return;
    }
    int p = 1;
    while (p < k) p *= 2;
    for (int i = tid; i < p; i += TT) {
        const u64 it = i < k ? sh.cand[i] : 0;
        sh.cand[MOST_K + i] = i < k ? (low - (it & low)) << 32 | it >> colbits : ~0ull;
    }
    __syncthreads();
    u64 *v = sh.cand + MOST_K;
    for (int size = 2; size <= p; size *= 2)
        for (int step = size / 2; step > 0; step /= 2) {
            for (int i = tid; i < p / 2; i += TT) {
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
        val[t * k + i] = Order<T>::value((uint32_t)v[i]);
    }
}

// Short rows and few entries of them (a router's choices): a warp per row, R consecutive columns a lane, so that of equal entries
// the lowest lane's is the lowest column's.  k times the warp takes the largest of its lanes' largest.
template <typename T, int R, bool LSE>
__global__ void __launch_bounds__(128)
top_short_kernel(int64_t nrows, int ncols, const T *__restrict__ xs, int64_t ldx, bool whole, int k, float c, float inv, int64_t *__restrict__ pos,
                 int64_t *__restrict__ crd, float *__restrict__ val, float *__restrict__ lse)
{
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
    uint32_t key[R], most = 0;
#pragma unroll
    for (int r = 0; r < R; r++) {
        key[r] = lane * R + r < ncols ? Order<T>::key(part.v[r]) : 0;
        most = max(most, key[r]);
    }
    int col = 0;
    uint32_t got = 0;                              // lane i: the i-th largest
    for (int i = 0; i < k; i++) {
        const uint32_t top = __reduce_max_sync(0xffffffffu, most);
        const int who = __ffs(__ballot_sync(0xffffffffu, most == top)) - 1;
        int at = 0;
        if (lane == who) {
            most = 0;
            bool found = false;
#pragma unroll
            for (int r = 0; r < R; r++) {
                if (!found && key[r] == top) {
                    found = true;
                    at = lane * R + r;
                    key[r] = 0;
                }
                most = max(most, key[r]);
            }
        }
        at = __shfl_sync(0xffffffffu, at, who);
        if (lane == i) {
            col = at;
            got = top;
        }
    }
    int place = 0;
    for (int i = 0; i < k; i++) place += __shfl_sync(0xffffffffu, col, i) < col;
    if (lane < k) {
        crd[t * k + place] = col;
        val[t * k + place] = Order<T>::value(got);
    }
    if (lane == 0) {
        pos[t] = t * k;
        if (t == nrows - 1) pos[nrows] = nrows * k;
    }
    if (LSE) {
        float m = MINUS_INF, s = 0.0f;
#pragma unroll
        for (int r = 0; r < R; r++) m = max_nan(m, to_float(part.v[r]));
        m = warp_max(m);
#pragma unroll
        for (int r = 0; r < R; r++) s += exp2_fast((to_float(part.v[r]) - m) * c);
        s = warp_sum(s);
        if (lane == 0) lse[t] = m == MINUS_INF ? m : fmaf(log2f(s), LN2, m * inv);
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
};

template <typename T, int R>
static void launch_short(const TopCall &a)
{
    const size_t piece = sizeof(T) * R < 16 ? sizeof(T) * R : 16;
    const bool whole = (uintptr_t)a.x % piece == 0 && a.ldx * (int64_t)sizeof(T) % (int64_t)piece == 0;
    const unsigned grid = (unsigned)ceil_div(a.nrows, 4);
    if (a.lse)
        top_short_kernel<T, R, true><<<grid, 128, 0, a.st>>>(a.nrows, a.ncols, (const T *)a.x, a.ldx, whole, a.k, a.c, a.inv, a.pos, a.crd, a.val, a.lse);
    else
        top_short_kernel<T, R, false><<<grid, 128, 0, a.st>>>(a.nrows, a.ncols, (const T *)a.x, a.ldx, whole, a.k, a.c, a.inv, a.pos, a.crd, a.val, a.lse);
}

template <typename T, bool LSE>
static int launch_long(const TopCall &a)
{
    constexpr int N = Granule<T>::N;
    const int all = (a.ncols + 2 * N - 2) / N;     // granules of a row, wherever it starts
    int ranks = 1, colbits = 1;
    while (ranks < MOST_RANKS && a.nrows * ranks <= sm_count() && all / ranks >= 2 * TU * TT) ranks *= 2;
    while ((1 << colbits) <= a.ncols) colbits++;
    const size_t smem = (size_t)STAGES * TU * TT * 16;
    if (a.nrows * ranks > 0x7fffffffLL) return fail("top_entries: more than 2^31 rows");
    return launch_cluster(top_kernel<T, LSE>, (unsigned)(a.nrows * ranks), ranks, TT, smem, a.st, a.nrows, a.ncols, (int)ceil_div(all, ranks),
                          (const T *)a.x, a.ldx, a.k, colbits, a.c, a.inv, a.pos, a.crd, a.val, a.lse);
}

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
    if (lse && !(*temperature > 0.0 && *temperature <= 1e30)) return fail("top_entries: temperature %g is not a positive number", *temperature);
    if ((uintptr_t)x % sizeof(T)) return fail("top_entries: an address that is not a multiple of the element's size");
    if (nrows == 0) {
        CB_CUDA(cudaMemsetAsync(pos, 0, sizeof(int64_t), st));
        return 0;
    }
    TopCall a = {nrows, (int)ncols, x, ldx, (int)k, 0.0f, 0.0f, pos, crd, val, lse, st};
    if (lse) {
        a.c = (float)(LOG2E_D / *temperature);
        a.inv = (float)(1.0 / *temperature);
    }
    if (ncols > 512 || k > 32) return lse ? launch_long<T, true>(a) : launch_long<T, false>(a);
    if (ncols <= 32) launch_short<T, 1>(a);
    else if (ncols <= 64) launch_short<T, 2>(a);
    else if (ncols <= 128) launch_short<T, 4>(a);
    else if (ncols <= 256) launch_short<T, 8>(a);
    else launch_short<T, 16>(a);
    CB_LAUNCH_CHECK();
    return 0;
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
