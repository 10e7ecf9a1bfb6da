// Rows of logits streamed once, by a CTA a row or a part of one (top.cu, logprob.cu): the ring of copies, and what is summed on the way.
#pragma once
#include "logits.cuh"

namespace cb200 {

static const int TT = 256, TW = TT / 32, TU = 4, STAGES = 3;

// What log_probs gives for each row beside the alternatives.
struct ProbCall {
    const int64_t *pos, *crd;
    float *values, *sums, *entropy;
};
template <typename T>
int top_log_probs(int64_t nrows, int ncols, const T *x, int64_t ldx, int k, float c, float inv, int64_t *pos, int64_t *crd, float *val, const ProbCall &probs,
                  cudaStream_t st);

#ifdef __CUDACC__
// A thread's way through a row, or a CTA's part of one: a ring of stages in shared memory, of which it copies and reads the same 16
// bytes each time, so the ring needs no barriers.
template <typename T>
struct Way {
    static constexpr int N = Granule<T>::N;
    uint4 *ring;                                   // STAGES * TU * TT
    const uint4 *from;                             // the row's granule 0
    int begin, end, all, off, ncols;               // the part, the row's granules, elements before the row, its columns
    const uint4 *next;
    int left, put, at;

    __device__ __forceinline__ int steps() const { return (end - begin + TU * TT - 1) / (TU * TT); }
    __device__ __forceinline__ void fetch()
    {
#pragma unroll
        for (int u = 0; u < TU; u++)
            if (u * TT < left) copy_granule(ring + (put * TU + u) * TT + threadIdx.x, next + u * TT);
        asm volatile("cp.async.commit_group;" ::: "memory");
        next += TU * TT;
        left -= TU * TT;
        put = put == STAGES - 1 ? 0 : put + 1;
    }
    __device__ __forceinline__ void start()
    {
        next = from + begin + threadIdx.x;
        left = end - begin - (int)threadIdx.x;
        put = at = 0;
#pragma unroll
        for (int i = 0; i < STAGES - 1; i++) fetch();
    }
    // the thread's granules of a step, TT apart; -inf where there is no row
    __device__ __forceinline__ Granule<T> *stage(int step)
    {
        fetch();
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        Granule<T> *mine = (Granule<T> *)(ring + at * TU * TT + threadIdx.x);
        at = at == STAGES - 1 ? 0 : at + 1;
        const int first = begin + step * TU * TT;
        if (first == 0 || first + TU * TT > min(end, all - 1)) {
#pragma unroll
            for (int u = 0; u < TU; u++) {
                const int i = first + threadIdx.x + u * TT;
                if (i == 0 || i >= all - 1 || i >= end) {
                    T *v = (T *)&mine[u * TT];
#pragma unroll
                    for (int e = 0; e < N; e++)
                        if (i >= end || i * N + e < off || i * N + e >= off + ncols) v[e] = from_float<T>(MINUS_INF);
                }
            }
        }
        return mine;
    }
    __device__ __forceinline__ int column(int step, int u, int e) const { return (begin + (step * TU + u) * TT + (int)threadIdx.x) * N + e - off; }
};

// A thread's sum of exp(x / temperature): its maximum, that times c, and two sums of 2^(x c - mc).
struct LogSum {
    float m, mc;
    float2 s;
    template <typename T>
    __device__ __forceinline__ void add(const Granule<T> (&g)[TU], typename Granule<T>::Most most, float c)
    {
        constexpr int N = Granule<T>::N;
        const float nm = max_nan(m, to_float(largest(most)));
        if (nm != m) {
            const float f = exp2_fast((m - nm) * c);
            s.x *= f;
            s.y *= f;
            m = nm;
            mc = m == MINUS_INF ? 0.0f : m * c;
        }
        if (fabsf(mc) < NEAR) {                    // what the rounding of mc does to s is below the rounding of the result, m c + log2(s)
#pragma unroll
            for (int u = 0; u < TU; u++) {
                float2 v[N / 2];
                g[u].unpack(v);
#pragma unroll
                for (int e = 0; e < N / 2; e++) {
                    const float2 d = fma2(v[e], make_float2(c, c), make_float2(-mc, -mc));
                    s = add2(s, make_float2(exp2_fast(d.x), exp2_fast(d.y)));
                }
            }
        } else {                                   // and NaN, and infinity
#pragma unroll
            for (int u = 0; u < TU; u++) {
                float v[N];
                g[u].unpack(v);
#pragma unroll
                for (int e = 0; e < N; e++) s.x += exp2_fast((v[e] - m) * c);
            }
        }
    }
};

// The log of a row's sum; with a maximum of +inf (no NaN then) s is of differences of infinities, and the sum is +inf.
__device__ __forceinline__ float log_of_sum(float m, float s, float inv) { return fabsf(m) == -MINUS_INF ? m : fmaf(log2f(s), LN2, m * inv); }

// The same with what a distribution is made of: sums of 2^d and, for the entropy, of d 2^d, d = (x - m) c in twos' powers.  Where m c is less than NEAR, d
// is x c - mc with mc the rounded product; `lacks` is what that is off by, a power of two that all terms share until it is taken out at the end.
template <bool ENTROPY>
struct ProbSum {
    float m, mc, lacks;
    bool near;
    float2 s, e;
    __device__ __forceinline__ void start()
    {
        m = MINUS_INF;
        mc = lacks = 0.0f;
        near = true;
        s = e = make_float2(0.0f, 0.0f);
    }
    __device__ __forceinline__ void raise(float nm, float c)
    {
        const float omc = mc, ol = lacks, om = m;
        const bool on = near;
        m = nm;
        mc = m == MINUS_INF ? 0.0f : m * c;
        near = fabsf(mc) < NEAR;
        lacks = near && m != MINUS_INF ? fmaf(m, c, -mc) : 0.0f;
        if (om == MINUS_INF) return;               // nothing summed so far
        const float d = on && near ? omc - mc : (om - m) * c - ol + lacks, f = exp2_fast(d);
        if (ENTROPY) {
            const float dd = fmaxf(d, -16384.0f);
            e.x = (e.x + s.x * dd) * f;
            e.y = (e.y + s.y * dd) * f;
        }
        s.x *= f;
        s.y *= f;
    }
    template <typename T, int U>
    __device__ __forceinline__ void add(const Granule<T> (&g)[U], typename Granule<T>::Most most, float c)
    {
        constexpr int N = Granule<T>::N;
        const float nm = max_nan(m, to_float(largest(most)));
        if (nm != m) raise(nm, c);
        if (near) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                float2 v[N / 2];
                g[u].unpack(v);
#pragma unroll
                for (int i = 0; i < N / 2; i++) {
                    const float2 d = fma2(v[i], make_float2(c, c), make_float2(-mc, -mc)), p = make_float2(exp2_fast(d.x), exp2_fast(d.y));
                    s = add2(s, p);
                    // a term of 0 adds 0, whatever its logarithm: that may be -inf
                    if (ENTROPY) e = fma2(p, make_float2(fmaxf(d.x, -16384.0f), fmaxf(d.y, -16384.0f)), e);
                }
            }
        } else {                                   // and NaN, and infinity
#pragma unroll
            for (int u = 0; u < U; u++) {
                float v[N];
                g[u].unpack(v);
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const float d = (v[i] - m) * c, p = exp2_fast(d);
                    s.x += p;
                    if (ENTROPY) e.x = fmaf(p, fmaxf(d, -16384.0f), e.x);
                }
            }
        }
    }
    // sums relative to m itself
    __device__ __forceinline__ void total(float &sum, float &ent) const
    {
        const float f = exp2_fast(-lacks);
        sum = (s.x + s.y) * f;
        ent = ENTROPY ? fmaf(-lacks, sum, (e.x + e.y) * f) : 0.0f;
    }
};

// What several threads, or CTAs, have of a row becomes relative to the largest of their maxima.
__device__ __forceinline__ void shift_to(float most, float m, float c, float &s, float &e)
{
    if (m == MINUS_INF) {
        s = e = 0.0f;
    } else if (m != most) {
        const float d = (m - most) * c, f = exp2_fast(d);
        e = (e + s * fmaxf(d, -16384.0f)) * f;
        s *= f;
    }
}

// A row's largest logit, and its sums: log s, and the entropy; the log probability of x.  A row of -inf has no distribution: its log probabilities are
// -inf, its entropy is 0.
struct RowProb {
    float m, log, entropy;
    __device__ __forceinline__ RowProb(float most, float s, float e) : m(most)
    {
        const float l2 = log2f(s);
        log = m == MINUS_INF ? 0.0f : l2 * LN2;
        entropy = m == MINUS_INF ? 0.0f : (l2 - e / s) * LN2;
    }
    __device__ __forceinline__ float of(float x, float inv) const { return m == MINUS_INF ? MINUS_INF : fmaf(x - m, inv, -log); }
};

// by `threads` threads, all of which have the row's sums
template <typename T>
__device__ __forceinline__ void give_probs(const ProbCall &a, int64_t t, const T *x, int ncols, const RowProb &p, float inv, int thread, int threads)
{
    if (thread == 0) {
        ((float2 *)a.sums)[t] = make_float2(p.m, p.log);
        if (a.entropy) a.entropy[t] = p.entropy;
    }
    for (int64_t e = a.pos[t] + thread; e < a.pos[t + 1]; e += threads) {
        const int64_t col = a.crd[e];
        a.values[e] = col < 0 || col >= ncols ? __int_as_float(0x7fffffff) : p.of(to_float(x[col]), inv);
    }
}
#endif

}  // namespace cb200
