// Log probabilities of given columns of rows of logits, the rows' entropies, and the gradient of both.  With u = x / temperature, m a row's largest logit,
// s = sum exp(u - m / temperature) and the pattern's entries (t, j):
//   value = (x_j - m) / temperature - log s,     entropy H = log s - sum exp(u - m / temperature) (u - m / temperature) / s
// and, with q = exp(value) of every column, d and h the gradients of the values and of the entropy that come in,
//   dx_j = (sum of d at j - q_j sum of d - h q_j (log q_j + H)) / temperature.
// What is kept from one to the other is m and log s, two f32 numbers: log s is small whatever the logits and the temperature are, so q is as good
// as the difference x - m.
//
// Forward: one pass; each thread has a maximum and sums of its own (rows.cuh), joined over the CTA and, where there are few rows, over a cluster that
// has cut the row.  Backward: one pass over pieces of rows, which no other CTA reads, so the gradient may take the place of the logits.
//
// Bound: HBM, and the exponential unit under the power cap: 4096 x 131072 bf16 with entropies 172 us alone, 190 in a row of passes (164 by the bytes; the unit is busy
// 77 % of the time at 1.86 GHz).  The gradient 390 (328 by the bytes).  Of short rows, a warp each, latency: 65536 x 256 bf16 25 us and the gradient 40 (5.4, 10.6),
// x 1000 39 and 77 (20, 40), in f32 75 and 143 (40, 80), 16384 x 2041 bf16 16 and 38 (10, 20).  The next longer rows are a CTA's each, which they do not
// fill: 65536 x 2048 bf16 434 and 302 (41, 82).  Every warp that works on a row's gradient looks at all of its entries: 512 x 131072 bf16 50 us with
// one entry a row, 53 with 32, 93 with 100, 478 with 1000.
#include "rows.cuh"

namespace cb200 {

template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(TT, 4)
prob_kernel(int ncols, int slice, const T *__restrict__ xs, int64_t ldx, float c, float inv, const ProbCall a)
{
    extern __shared__ __align__(128) uint4 ring[];  // a warp reads 512 bytes at a time: from a line on, or a fifth line takes an eighth more time
    __shared__ float room[3 * TW], told[3 * MOST_CLUSTER];
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
    if (ranks > 1) cluster_arrive_relaxed();       // only to say that it is there
    ProbSum<ENTROPY> sum;
    sum.start();
    way.start();
    const int steps = way.steps();
    for (int step = 0; step < steps; step++) {
        const Granule<T> *mine = way.stage(step);
        Granule<T> g[TU];
#pragma unroll
        for (int u = 0; u < TU; u++) g[u] = mine[u * TT];
        sum.add(g, most_of(most_of(g[0].most(), g[1].most()), most_of(g[2].most(), g[3].most())), c);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    float q[2], r[1] = {sum.m};
    sum.total(q[0], q[1]);
    cta_reduce<1, TW, true>(r, room);
    shift_to(r[0], sum.m, c, q[0], q[1]);
    cta_reduce<2, TW, false>(q, room + TW);
    float m = r[0], s = q[0], ent = q[1];
    if (ranks > 1) {
        cluster_wait();
        if (tid < (int)ranks) {
            store_peer(&told[3 * rank], tid, m);
            store_peer(&told[3 * rank + 1], tid, s);
            store_peer(&told[3 * rank + 2], tid, ent);
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (rank != 0) return;
        m = told[0];
        for (unsigned i = 1; i < ranks; i++) m = max_nan(m, told[3 * i]);
        s = ent = 0.0f;
        for (unsigned i = 0; i < ranks; i++) {
            float os = told[3 * i + 1], oe = told[3 * i + 2];
            shift_to(m, told[3 * i], c, os, oe);
            s += os;
            ent += oe;
        }
    }
    give_probs(a, t, x, ncols, RowProb(m, s, ent), inv, tid, TT);
}

// A row's granules to registers, lane by lane; -inf where there is no row.
template <typename T, int G>
__device__ __forceinline__ void load_row(Granule<T> (&g)[G], const T *x, int ncols, int lane)
{
    constexpr int N = Granule<T>::N;
    const uint4 *from = (const uint4 *)((uintptr_t)x & ~(uintptr_t)15);
    const int off = (int)((uintptr_t)x & 15) / (int)sizeof(T), all = (off + ncols + N - 1) / N;
#pragma unroll
    for (int i = 0; i < G; i++) {
        const int at = i * 32 + lane;
        g[i] = Granule<T>::least();
        if (at < all) {
            g[i].w = from[at];
            if (at == 0 || at == all - 1) {
                T *v = (T *)&g[i];
#pragma unroll
                for (int k = 0; k < N; k++)
                    if (at * N + k < off || at * N + k >= off + ncols) v[k] = from_float<T>(MINUS_INF);
            }
        }
    }
}

// Short rows: a warp each.
template <typename T, int G, bool ENTROPY>
__global__ void __launch_bounds__(128)
prob_short_kernel(int64_t nrows, int ncols, const T *__restrict__ xs, int64_t ldx, float c, float inv, const ProbCall a)
{
    const int lane = threadIdx.x & 31;
    const int64_t t = ((int64_t)blockIdx.x * 128 + threadIdx.x) >> 5;
    if (t >= nrows) return;
    const T *x = xs + t * ldx;
    Granule<T> g[G];
    load_row<T, G>(g, x, ncols, lane);
    typename Granule<T>::Most most = g[0].most();
#pragma unroll
    for (int i = 1; i < G; i++) most = most_of(most, g[i].most());
    ProbSum<ENTROPY> sum;
    sum.start();
    sum.add(g, most, c);
    float s, ent;
    sum.total(s, ent);
    const float m = warp_max(sum.m);
    shift_to(m, sum.m, c, s, ent);
    s = warp_sum(s);
    if (ENTROPY) ent = warp_sum(ent);
    give_probs(a, t, x, ncols, RowProb(m, s, ent), inv, lane, 32);
}

struct ProbGrad {
    int64_t nrows;
    int ncols;
    const int64_t *pos, *crd;
    const float *sums, *values, *entropy, *by_entropy;           // values: their gradients; by_entropy: the entropies' (null: none)
    int64_t ldx, ldg;
    float c, inv;
};

// A row's terms: dx = q (a + b log2 q) where no entry is, and exponents.
template <bool ENTROPY>
struct GradRow {
    float c, m, mc, less, a, b;
    bool near, none, zero;
    __device__ __forceinline__ GradRow(const ProbGrad &p, float2 row, float h, float entropy, float sum)
    {
        c = p.c;
        m = row.x;
        none = m == MINUS_INF;
        mc = none ? 0.0f : m * c;
        near = fabsf(mc) < NEAR;
        less = row.y * LOG2E + (near && !none ? fmaf(m, c, -mc) : 0.0f);             // what the exponent is beyond log2 q
        a = -p.inv * (sum + (ENTROPY && h != 0.0f ? h * entropy : 0.0f));
        b = ENTROPY ? -p.inv * LN2 * h : 0.0f;
        zero = none || (sum == 0.0f && h == 0.0f);
    }
    __device__ __forceinline__ float2 from_exponent(float2 d) const
    {
        d = add2(d, make_float2(-less, -less));
        const float2 q = make_float2(exp2_fast(d.x), exp2_fast(d.y));
        if (!ENTROPY) return mul2(q, make_float2(a, a));
        // a q of 0 gives 0, whatever its logarithm: that may be -inf
        return mul2(q, fma2(make_float2(fmaxf(d.x, -16384.0f), fmaxf(d.y, -16384.0f)), make_float2(b, b), make_float2(a, a)));
    }
    template <int H>
    __device__ __forceinline__ void all(float2 (&v)[H]) const
    {
        if (zero) {
#pragma unroll
            for (int k = 0; k < H; k++) v[k] = make_float2(0.0f, 0.0f);
        } else if (near) {
#pragma unroll
            for (int k = 0; k < H; k++) v[k] = from_exponent(fma2(v[k], make_float2(c, c), make_float2(-mc, -mc)));
        } else {
#pragma unroll
            for (int k = 0; k < H; k++) v[k] = from_exponent(make_float2((v[k].x - m) * c, (v[k].y - m) * c));
        }
    }
};

template <typename T>
__device__ __forceinline__ void put_granule(T *g, int col, int ncols, bool alike, const float2 (&v)[Granule<T>::N / 2])
{
    constexpr int N = Granule<T>::N;
    Granule<T> out;
    out.pack(v);
    if (alike && col >= 0 && col + N <= ncols) {
        *(uint4 *)(g + col) = out.w;
    } else {
#pragma unroll
        for (int k = 0; k < N; k++)
            if (col + k >= 0 && col + k < ncols) g[col + k] = ((const T *)&out)[k];
    }
}

// A lane's share of a row's entries, 32 at a time: their sum, by every warp.
__device__ __forceinline__ float sum_entries(const float *values, int64_t lo, int64_t hi, int lane)
{
    float sum = 0.0f;
    for (int64_t e = lo + lane; e < hi; e += 32) sum += values[e];
    return warp_sum(sum);
}
// The entries among a warp's granules, 32 at a time, a lane each.  Granule i of a lane begins at column col0 + (i * stride + first + lane) * N.
struct Hits {
    int granule, at;                 // negative: not one of the warp's
    float d;
    template <int G, int N>
    __device__ __forceinline__ void load(const ProbGrad &p, int64_t e, int64_t hi, int col0, int stride, int first)
    {
        granule = -1;
        if (e < hi) {
            const int64_t col = p.crd[e], j = col - col0;
            if (col >= 0 && col < p.ncols && j >= 0 && j < (int64_t)G * stride * N) {
                const int g = (int)j / N;
                if ((g % stride & ~31) == first) {
                    granule = g;
                    at = (int)j % N;
                    d = p.values[e] * p.inv;
                }
            }
        }
    }
    // those of granules `i`
    template <int N>
    __device__ __forceinline__ void add(int i, int stride, int first, int lane, float2 (&v)[N / 2]) const
    {
        for (unsigned on = __ballot_sync(0xffffffffu, granule >= 0 && granule / stride == i); on; on &= on - 1) {
            const int who = __ffs(on) - 1, g = __shfl_sync(0xffffffffu, granule, who), k = __shfl_sync(0xffffffffu, at, who);
            const float x = __shfl_sync(0xffffffffu, d, who);
            const int to = g % stride - first == lane ? k : -1;
            // no branch: the granule stays in registers
#pragma unroll
            for (int n = 0; n < N / 2; n++) {
                v[n].x += to == 2 * n ? x : 0.0f;
                v[n].y += to == 2 * n + 1 ? x : 0.0f;
            }
        }
    }
};
// Computes and stores a thread's granules: `left` of them, stride apart, are the row's.
template <typename T, int G, bool ENTROPY>
__device__ __forceinline__ void give_gradients(const ProbGrad &p, const GradRow<ENTROPY> &row, const Granule<T> (&in)[G], T *g, bool alike, int64_t lo, int64_t hi, int col0,
                                               int stride, int place, int left)
{
    constexpr int N = Granule<T>::N;
    const int lane = threadIdx.x & 31, first = place & ~31;
    Hits hits;
    hits.load<G, N>(p, lo + lane, hi, col0, stride, first);
    const bool some = !row.none && __any_sync(0xffffffffu, hits.granule >= 0), more = !row.none && hi - lo > 32;
#pragma unroll
    for (int i = 0; i < G; i++) {
        float2 v[N / 2];
        in[i].unpack(v);
        row.all(v);
        if (some) hits.add<N>(i, stride, first, lane, v);
        if (more)
            for (int64_t e = lo + 32; e < hi; e += 32) {
                Hits h;
                h.load<G, N>(p, e + lane, hi, col0, stride, first);
                h.add<N>(i, stride, first, lane, v);
            }
        if (i * stride + place < left) put_granule<T>(g, col0 + (i * stride + place) * N, p.ncols, alike, v);
    }
}

// A piece of a row a CTA, G granules a thread: 128 bytes of f32, 64 of 16 bits.  No barrier: a warp finds its granules' entries itself.
static const int GT = 256;
template <typename T>
constexpr int grad_granules() { return sizeof(T) == 4 ? 8 : 4; }
template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(GT)
prob_grad_kernel(const ProbGrad p, int pieces, const T *xs, T *grad)
{
    constexpr int N = Granule<T>::N, G = grad_granules<T>();
    const int tid = threadIdx.x, lane = tid & 31, piece = blockIdx.x % pieces;
    const int64_t t = blockIdx.x / pieces;
    const T *x = xs + t * p.ldx;
    T *g = grad + t * p.ldg;
    const uint4 *from = (const uint4 *)((uintptr_t)x & ~(uintptr_t)15) + piece * GT * G;
    const int off = (int)((uintptr_t)x & 15) / (int)sizeof(T), left = (off + p.ncols + N - 1) / N - piece * GT * G, col0 = piece * GT * G * N - off;
    const bool alike = (((uintptr_t)g ^ (uintptr_t)x) & 15) == 0;
    Granule<T> in[G];
#pragma unroll
    for (int i = 0; i < G; i++) {
        in[i].w = make_uint4(0, 0, 0, 0);
        if (i * GT + tid < left) in[i].w = from[i * GT + tid];
    }
    const int64_t lo = p.pos[t], hi = p.pos[t + 1];
    const float2 kept = ((const float2 *)p.sums)[t];
    const float h = ENTROPY ? p.by_entropy[t] : 0.0f, ent = ENTROPY ? p.entropy[t] : 0.0f;
    const GradRow<ENTROPY> row(p, kept, h, ent, sum_entries(p.values, lo, hi, lane));
    give_gradients<T, G, ENTROPY>(p, row, in, g, alike, lo, hi, col0, GT, tid, left);
}

// Short rows: a warp each, which has the whole row in registers.
template <typename T, int G, bool ENTROPY>
__global__ void __launch_bounds__(128)
prob_grad_short_kernel(const ProbGrad p, const T *xs, T *grad)
{
    constexpr int N = Granule<T>::N;
    const int lane = threadIdx.x & 31;
    const int64_t t = ((int64_t)blockIdx.x * 128 + threadIdx.x) >> 5;
    if (t >= p.nrows) return;
    const T *x = xs + t * p.ldx;
    T *g = grad + t * p.ldg;
    Granule<T> in[G];
    load_row<T, G>(in, x, p.ncols, lane);
    const int64_t lo = p.pos[t], hi = p.pos[t + 1];
    const int off = (int)((uintptr_t)x & 15) / (int)sizeof(T);
    const bool alike = (((uintptr_t)g ^ (uintptr_t)x) & 15) == 0;
    const float h = ENTROPY ? p.by_entropy[t] : 0.0f, ent = ENTROPY ? p.entropy[t] : 0.0f;
    const GradRow<ENTROPY> row(p, ((const float2 *)p.sums)[t], h, ent, sum_entries(p.values, lo, hi, lane));
    give_gradients<T, G, ENTROPY>(p, row, in, g, alike, lo, hi, -off, 32, lane, 32 * G);
}

template <typename T>
static int check_logits(const char *what, int64_t nrows, int64_t ncols, const void *x, int64_t ldx, const double *temperature, const float *sums)
{
    if (nrows < 0 || ncols <= 0 || ncols >= 1LL << 30) return fail("%s: %lld rows of %lld columns", what, (long long)nrows, (long long)ncols);
    if (ldx < ncols) return fail("%s: leading dimension smaller than the number of columns", what);
    if (nrows > 0x7fffffffLL / MOST_CLUSTER) return fail("%s: more than 2^28 rows", what);
    if (!temperature_fits(*temperature)) return fail("%s: temperature %g is not a number of 1e-38 to 1e30", what, *temperature);
    if ((uintptr_t)x % sizeof(T)) return fail("%s: an address that is not a multiple of the element's size", what);
    if ((uintptr_t)sums % sizeof(float2)) return fail("%s: sums at an address that is not a multiple of 8 bytes", what);
    return 0;
}

// granules a lane that take any row of ncols columns; 0: the row is not short
template <typename T>
static int lane_granules(int64_t ncols)
{
    const int64_t all = (ncols + 2 * Granule<T>::N - 2) / Granule<T>::N;
    return all <= 32 ? 1 : all <= 64 ? 2 : all <= 128 ? 4 : all <= 256 ? 8 : 0;
}

template <typename T, bool ENTROPY>
static int launch_probs(int64_t nrows, int ncols, const T *x, int64_t ldx, float c, float inv, const ProbCall &a, cudaStream_t st)
{
    const unsigned grid = (unsigned)ceil_div(nrows, 4);
    switch (lane_granules<T>(ncols)) {
    case 1: prob_short_kernel<T, 1, ENTROPY><<<grid, 128, 0, st>>>(nrows, ncols, x, ldx, c, inv, a); break;
    case 2: prob_short_kernel<T, 2, ENTROPY><<<grid, 128, 0, st>>>(nrows, ncols, x, ldx, c, inv, a); break;
    case 4: prob_short_kernel<T, 4, ENTROPY><<<grid, 128, 0, st>>>(nrows, ncols, x, ldx, c, inv, a); break;
    case 8: prob_short_kernel<T, 8, ENTROPY><<<grid, 128, 0, st>>>(nrows, ncols, x, ldx, c, inv, a); break;
    default: {
        const int all = (ncols + 2 * Granule<T>::N - 2) / Granule<T>::N;
        int ranks = 1;
        while (ranks < MOST_CLUSTER && nrows * ranks <= sm_count() && all / ranks >= 2 * TT) ranks *= 2;
        const size_t smem = (size_t)STAGES * TU * TT * 16;
        return launch_cluster(prob_kernel<T, ENTROPY>, (unsigned)(nrows * ranks), ranks, TT, smem, smem, st, ncols, (int)ceil_div(all, ranks), x, ldx, c, inv, a);
    }
    }
    CB_LAUNCH_CHECK();
    return 0;
}

template <typename T>
static int log_probs(int64_t nrows, int64_t ncols, const int64_t *pos, const int64_t *crd, const void *x, int64_t ldx, const double *temperature, float *values,
                     float *sums, float *entropy, int64_t k, int64_t *best_pos, int64_t *best_crd, float *best_val, cudaStream_t st)
{
    clear_error();
    CB_TRY(check_logits<T>("log_probs", nrows, ncols, x, ldx, temperature, sums));
    if (k < 0 || k > ncols || k > 1024) return fail("log_probs: %lld alternatives a row; 0 to 1024, and no more than a row has columns", (long long)k);
    if (nrows == 0) {
        if (k) CB_CUDA(cudaMemsetAsync(best_pos, 0, sizeof(int64_t), st));
        return 0;
    }
    const ProbCall a = {pos, crd, values, sums, entropy};
    const float c = (float)(LOG2E_D / *temperature), inv = (float)(1.0 / *temperature);
    if (k) return top_log_probs<T>(nrows, (int)ncols, (const T *)x, ldx, (int)k, c, inv, best_pos, best_crd, best_val, a, st);
    return entropy ? launch_probs<T, true>(nrows, (int)ncols, (const T *)x, ldx, c, inv, a, st)
                   : launch_probs<T, false>(nrows, (int)ncols, (const T *)x, ldx, c, inv, a, st);
}

template <typename T, bool ENTROPY>
static int launch_grad(const ProbGrad &p, const T *x, T *grad, cudaStream_t st)
{
    const unsigned grid = (unsigned)ceil_div(p.nrows, 4);
    switch (lane_granules<T>(p.ncols)) {
    case 1: prob_grad_short_kernel<T, 1, ENTROPY><<<grid, 128, 0, st>>>(p, x, grad); break;
    case 2: prob_grad_short_kernel<T, 2, ENTROPY><<<grid, 128, 0, st>>>(p, x, grad); break;
    case 4: prob_grad_short_kernel<T, 4, ENTROPY><<<grid, 128, 0, st>>>(p, x, grad); break;
    case 8: prob_grad_short_kernel<T, 8, ENTROPY><<<grid, 128, 0, st>>>(p, x, grad); break;
    default: {
        const int64_t pieces = ceil_div((p.ncols + 2 * Granule<T>::N - 2) / Granule<T>::N, GT * grad_granules<T>());
        if (pieces * p.nrows > 0x7fffffffLL) return fail("log_probs_grad: more than 2^31 pieces of rows");
        prob_grad_kernel<T, ENTROPY><<<(unsigned)(pieces * p.nrows), GT, 0, st>>>(p, (int)pieces, x, grad);
    }
    }
    CB_LAUNCH_CHECK();
    return 0;
}

template <typename T>
static int log_probs_grad(int64_t nrows, int64_t ncols, const int64_t *pos, const int64_t *crd, const void *x, int64_t ldx, const double *temperature,
                          const float *sums, const float *values, const float *entropy, const float *by_entropy, void *grad, int64_t ldg, cudaStream_t st)
{
    clear_error();
    CB_TRY(check_logits<T>("log_probs_grad", nrows, ncols, x, ldx, temperature, sums));
    if (ldg < ncols) return fail("log_probs_grad: leading dimension smaller than the number of columns");
    if ((uintptr_t)grad % sizeof(T)) return fail("log_probs_grad: an address that is not a multiple of the element's size");
    if (by_entropy && !entropy) return fail("log_probs_grad: the entropies' gradients need the entropies");
    if (nrows == 0) return 0;
    const ProbGrad p = {nrows, (int)ncols, pos, crd, sums, values, entropy, by_entropy, ldx, ldg, (float)(LOG2E_D / *temperature), (float)(1.0 / *temperature)};
    return by_entropy ? launch_grad<T, true>(p, (const T *)x, (T *)grad, st) : launch_grad<T, false>(p, (const T *)x, (T *)grad, st);
}

}  // namespace cb200

#define LOG_PROBS(suffix, T)                                                                                                                           \
    extern "C" int32_t comet_b200_dev_log_probs_##suffix##_i64(int64_t nrows, int64_t ncols, const int64_t *pos, const int64_t *crd, const void *x,    \
                                                               int64_t ldx, const double *temperature, float *values, float *sums, float *entropy,     \
                                                               int64_t k, int64_t *best_pos, int64_t *best_crd, float *best_val, void *stream)         \
    {                                                                                                                                                  \
        return cb200::log_probs<T>(nrows, ncols, pos, crd, x, ldx, temperature, values, sums, entropy, k, best_pos, best_crd, best_val,                \
                                   (cudaStream_t)stream);                                                                                              \
    }                                                                                                                                                  \
    extern "C" int32_t comet_b200_dev_log_probs_grad_##suffix##_i64(                                                                                   \
        int64_t nrows, int64_t ncols, const int64_t *pos, const int64_t *crd, const void *x, int64_t ldx, const double *temperature,                    \
        const float *sums, const float *d_values, const float *entropy, const float *d_entropy, void *grad, int64_t ldg, void *stream)                 \
    {                                                                                                                                                  \
        return cb200::log_probs_grad<T>(nrows, ncols, pos, crd, x, ldx, temperature, sums, d_values, entropy, d_entropy, grad, ldg,                    \
                                        (cudaStream_t)stream);                                                                                         \
    }
LOG_PROBS(bf16, __nv_bfloat16)
LOG_PROBS(f16, __half)
LOG_PROBS(f32, float)
