// The k largest entries of each row of a dense matrix as a CSR matrix, columns ascending, and the log of the sum of the row's
// exp(x / temperature).  Equal entries: the lower column; NaN is above all numbers; -0 equals 0.
//
// An entry is compared as 64 bits: its value in an order-preserving code, then the complement of its column, so no two are
// equal and the k largest are always the same k.
// A CTA streams its row once.  The first step's 1024 groups of 16 bytes have a largest entry each, and the k-th largest of
// those is a bound that k entries reach, so few entries of the rest of the row pass it; they are kept in shared memory.
// Where they do not fit, the k largest so far are kept and the k-th of them is the new bound.
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

static const int TT = 256, TU = 4, MOST_K = 1024, ROOM = 2048;

__device__ __forceinline__ uint32_t order_key(float v)
{
    const uint32_t u = __float_as_uint(v + 0.0f);
    return v != v ? 0xffffffffu : u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k == 0xffffffffu ? 0x7fffffffu : k ^ ((int32_t)k < 0 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ unsigned long long entry(float v, uint32_t col) { return (unsigned long long)order_key(v) << 32 | (0xffffffffu - col); }

struct TopShared {
    unsigned long long cand[ROOM];
    unsigned long long sel[MOST_K];
    int hist[256];
    int digit, left, exact;
    int count;
    float room[2 * TT / 32];
};

// The least number that exactly k of cand[0..n) reach (from bit `lowest` up: at least k).  k <= n.
__device__ unsigned long long kth_largest(TopShared &sh, int n, int k, int lowest)
{
    unsigned long long prefix = 0;
    int left = k;
    if (n <= k) return 0;
    for (int shift = 56; shift >= lowest; shift -= 8) {
        const unsigned long long mask = shift == 56 ? 0 : ~0ull << (shift + 8);
        sh.hist[threadIdx.x] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += TT) {
            const unsigned long long c = sh.cand[i];
            if (((c ^ prefix) & mask) == 0) atomicAdd(&sh.hist[(int)(c >> shift) & 255], 1);
        }
        __syncthreads();
        if (threadIdx.x < 32) {                    // lane l: the eight digits from 255 - 8 l down
            int own[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) sum += own[i] = sh.hist[255 - 8 * threadIdx.x - i];
            int before = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, before, o);
                if ((int)threadIdx.x >= o) before += v;
            }
            before -= sum;
            if (before < left && left <= before + sum) {
                bool found = false;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (!found && left <= before + own[i]) {
                        found = true;
                        sh.digit = 255 - 8 * threadIdx.x - i;
                        sh.left = left - before;
                        sh.exact = left - before == own[i];
                    }
                    before += own[i];
                }
            }
        }
        __syncthreads();
        prefix |= (unsigned long long)sh.digit << shift;
        left = sh.left;
        if (sh.exact) break;
    }
    return prefix;
}

// The k largest of cand[0..n) to the front, in any order; returns the least of them (or a number that only they reach).
__device__ unsigned long long keep_largest(TopShared &sh, int n, int k)
{
    const unsigned long long least = kth_largest(sh, n, k, 0);
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += TT) {
        const unsigned long long c = sh.cand[i];
        if (c >= least) sh.sel[atomicAdd(&sh.count, 1)] = c;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < min(n, k); i += TT) sh.cand[i] = sh.sel[i];
    __syncthreads();
    return least;
}

template <typename T, bool LSE>
__global__ void __launch_bounds__(TT)
top_kernel(int64_t nrows, int ncols, const T *__restrict__ xs, int64_t ldx, int k, float c, float inv, int64_t *__restrict__ pos, int64_t *__restrict__ crd,
           float *__restrict__ val, float *__restrict__ lse)
{
    constexpr int N = Granule<T>::N;
    __shared__ TopShared sh;
    const int tid = threadIdx.x;
    const int64_t t = blockIdx.x;
    const T *x = xs + t * ldx;
    const int off = (int)((uintptr_t)x & 15) / (int)sizeof(T), all = (off + ncols + N - 1) / N;
    const uint4 *from = (const uint4 *)((uintptr_t)x & ~(uintptr_t)15);
    if (tid == 0) sh.count = 0;
    __syncthreads();
    unsigned long long bound = 0;                  // an entry has to be larger
    float m = MINUS_INF, s = 0.0f;
    for (int g0 = 0; g0 < all; g0 += TT * TU) {
        Granule<T> g[TU];
        float gm[TU];
#pragma unroll
        for (int u = 0; u < TU; u++) {
            const int i = g0 + u * TT + tid;
            if (i < all) g[u].w = __ldcs(from + i);
        }
#pragma unroll
        for (int u = 0; u < TU; u++) {
            const int i = g0 + u * TT + tid;
            if (i == 0 || i >= all - 1) {          // entries before and behind the row
                float v[N];
                g[u].unpack(v);
#pragma unroll
                for (int e = 0; e < N; e++)
                    if (i >= all || i * N + e < off || i * N + e >= off + ncols) v[e] = MINUS_INF;
                g[u].pack(v);
            }
            gm[u] = granule_max(g[u]);
            if (LSE) {
                const float nm = max_nan(m, gm[u]);
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
        if (g0 == 0 && all > TT) {
#pragma unroll
            for (int u = 0; u < TU; u++) sh.cand[u * TT + tid] = (unsigned long long)order_key(gm[u]) << 32;
            __syncthreads();
            bound = kth_largest(sh, TT * TU, k, 32);
            __syncthreads();
        }
        unsigned pending = 0;
        auto look = [&](bool put) {
#pragma unroll
            for (int u = 0; u < TU; u++) {
                if (put ? !(pending >> (u * N) & ((1u << N) - 1)) : (unsigned long long)order_key(gm[u]) << 32 < (bound & ~0xffffffffull)) continue;
                float v[N];
                g[u].unpack(v);
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const int col = (g0 + u * TT + tid) * N + e - off;
                    const unsigned long long it = entry(v[e], (uint32_t)col);
                    const unsigned bit = 1u << (u * N + e);
                    if (!put) {
                        if (it > bound && col >= 0 && col < ncols) pending |= bit;
                    } else if (pending & bit) {
                        const int at = atomicAdd(&sh.count, 1);
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
            if (!__syncthreads_or(pending != 0)) break;
            const unsigned long long least = keep_largest(sh, ROOM, k);
            if (least - 1 > bound) bound = least - 1;
            if (pending) {                         // of those that found no room, the ones that are still large enough
                const unsigned without = pending;
                pending = 0;
                look(false);
                pending &= without;
            }
            if (tid == 0) sh.count = k;
            __syncthreads();
        }
    }
    __syncthreads();
    keep_largest(sh, sh.count, k);
    // by column, ascending
    int p = 1;
    while (p < k) p *= 2;
    for (int i = tid; i < p; i += TT) {
        const unsigned long long v = i < k ? sh.cand[i] : 0;
        sh.sel[i] = (unsigned long long)(0xffffffffu - (uint32_t)v) << 32 | v >> 32;     // v = 0: behind all columns
    }
    __syncthreads();
    for (int size = 2; size <= p; size *= 2)
        for (int step = size / 2; step > 0; step /= 2) {
            for (int i = tid; i < p / 2; i += TT) {
                const int lo = i / step * step * 2 + i % step, hi = lo + step;
                const unsigned long long a = sh.sel[lo], b = sh.sel[hi];
                if ((a > b) == ((lo & size) == 0)) {
                    sh.sel[lo] = b;
                    sh.sel[hi] = a;
                }
            }
            __syncthreads();
        }
    for (int i = tid; i < k; i += TT) {
        crd[t * k + i] = (int64_t)(sh.sel[i] >> 32);
        val[t * k + i] = key_value((uint32_t)sh.sel[i]);
    }
    if (tid == 0) {
        pos[t] = t * k;
        if (t == nrows - 1) pos[nrows] = nrows * k;
    }
    if (LSE) {
        float r[1] = {m}, q[1];
        cta_reduce<1, TT / 32, true>(r, sh.room);
        q[0] = m == MINUS_INF ? 0.0f : s * exp2_fast((m - r[0]) * c);
        cta_reduce<1, TT / 32, false>(q, sh.room + TT / 32);
        if (tid == 0) lse[t] = r[0] == MINUS_INF ? r[0] : fmaf(log2f(q[0]), LN2, r[0] * inv);
    }
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
    const float c = lse ? (float)(LOG2E_D / *temperature) : 0.0f, inv = lse ? (float)(1.0 / *temperature) : 0.0f;
    if (lse)
        top_kernel<T, true><<<(unsigned)nrows, TT, 0, st>>>(nrows, (int)ncols, (const T *)x, ldx, (int)k, c, inv, pos, crd, val, lse);
    else
        top_kernel<T, false><<<(unsigned)nrows, TT, 0, st>>>(nrows, (int)ncols, (const T *)x, ldx, (int)k, c, inv, pos, crd, val, lse);
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
