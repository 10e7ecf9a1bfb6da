// Distillation from a teacher's top logits: the teacher is a CSR matrix S (rows tokens, columns the vocabulary) of the logits
// it has listed, the student a dense matrix X.  With c = log2(e) / temperature, q = softmax(X / temperature) and
//   p_j = exp(z_j / temperature) / sum over the row's entries                      (without lse)
//   p_j = exp(z_j / temperature - lse), left = max(0, 1 - sum p)                   (with lse: the rest is one outcome)
// a row's loss is sum p (log p - log q) [+ left (log left - log q_rest), q_rest = the sum of q where nothing is stored], and
//   d loss / d x_j = (q_j - p_j) / temperature where an entry is stored, q_j (1 - left / q_rest) / temperature elsewhere.
// q_rest is a sum of its own, not 1 minus the rest: where the teacher lists nearly all, the difference would have no digits left.
//
// A cluster of CTAs takes a row: each has its part of the row copied into shared memory (16 bytes a copy, no registers), so
// X is read from HBM once, and the maximum, the sums and the gradient are three passes over shared memory.  What the CTAs of
// a row have to tell each other are five floats, written into each other's shared memory.
//
// Bound: HBM, the bytes of X and of the gradient.
#include "logits.cuh"

namespace cb200 {

static const int DT = 256, DW = DT / 32;
static const int MOST_SLICE = 192 * 1024;          // bytes of a row in one CTA

struct DistillArgs {
    int64_t nrows;
    int ncols, slice;            // granules per CTA
    const int64_t *pos, *crd;
    const void *val;
    const float *lse, *weight;
    const void *x;
    int64_t ldx;
    void *grad;
    int64_t ldg;
    float c, by, scale;          // log2(e) / temperature, scale / temperature
    float *rows, *loss;
    unsigned *counter;
};

// what a CTA tells the others of its row: the maximum of its part, sums of 2^((x - maximum) c) of elements that are not
// stored and of those that are, of p's weights and of p's weights times (x - maximum) c
struct Told {
    float m, others, stored, p, pu;
};

template <typename T, typename TV, bool REST, bool GRAD>
__global__ void __launch_bounds__(DT)
distill_kernel(const DistillArgs a)
{
    constexpr int N = Granule<T>::N;
    extern __shared__ uint4 dyn[];
    __shared__ float room[6 * DW], room2[2 * DW];
    __shared__ Told told[MOST_CLUSTER];
    __shared__ bool last;
    const int tid = threadIdx.x;
    const unsigned rank = cluster_rank(), ranks = cluster_size();
    const int64_t t = blockIdx.x / ranks, lo = a.pos[t], hi = a.pos[t + 1];
    const float w = a.weight ? a.weight[t] : 1.0f;
    const T *x = (const T *)a.x + t * a.ldx;
    const TV *z = (const TV *)a.val;
    // the row's granules, and this CTA's; element e of them is column e - off + first * N
    const int off = (int)((uintptr_t)x & 15) / (int)sizeof(T);
    const int all = (off + a.ncols + N - 1) / N, first = min((int)rank * a.slice, all), n = min(a.slice, all - first);
    const int col0 = first * N - off;              // the column of this CTA's element 0; negative if that lies before the row
    uint4 *part = dyn;
    uint32_t *bits = (uint32_t *)(dyn + a.slice);  // a bit per element: stored
    T *elem = (T *)part;

    float m[2] = {MINUS_INF, MINUS_INF};
    cluster_arrive();
    if (lo < hi && w != 0.0f) {
        const uint4 *from = (const uint4 *)((uintptr_t)x & ~(uintptr_t)15) + first;
        for (int i = tid; i < n; i += DT) copy_granule(part + i, from + i);
        if (REST)
            for (int i = tid; i < (n * N + 31) / 32; i += DT) bits[i] = 0;
        for (int64_t e = lo + tid; e < hi; e += DT) m[1] = max_nan(m[1], (float)z[e]);
        wait_copies();
        for (int i = tid; i < n; i += DT) {
            if (i == 0 || i == n - 1)              // elements before and behind the row
                for (int k = 0; k < N; k++)
                    if (col0 + i * N + k < 0 || col0 + i * N + k >= a.ncols) elem[i * N + k] = from_float<T>(MINUS_INF);
            m[0] = max_nan(m[0], to_float(largest(((const Granule<T> *)(part + i))->most())));
        }
    }
    cta_reduce<2, DW, true>(m, room2);
    const bool counts = m[1] != MINUS_INF;         // the row stores something, and its weight is not 0
    float s[6] = {0, 0, 0, 0, 0, 0};
    const float mx = m[0] == MINUS_INF ? 0.0f : m[0];
    if (counts) {
        if (REST) {
            for (int64_t e = lo + tid; e < hi; e += DT) {
                const int64_t j = a.crd[e] - col0;
                if (j >= 0 && j < (int64_t)n * N) atomicOr(&bits[j >> 5], 1u << (j & 31));
            }
            __syncthreads();
        }
        for (int i = tid; i < n; i += DT) {
            float v[N];
            ((const Granule<T> *)(part + i))->unpack(v);
            unsigned skip = 0;
            if (REST) skip = N == 8 ? ((const uint8_t *)bits)[i] : ((const uint8_t *)bits)[i >> 1] >> ((i & 1) * 4);
#pragma unroll
            for (int k = 0; k < N; k++) {
                const float q = exp2_fast((v[k] - mx) * a.c);
                if (!REST || !(skip >> k & 1)) s[0] += q;
            }
        }
        const float zref = REST ? a.lse[t] * LOG2E : m[1];
        for (int64_t e = lo + tid; e < hi; e += DT) {
            const int64_t col = a.crd[e], j = col - col0;
            const float lz = REST ? fmaf((float)z[e], a.c, -zref) : ((float)z[e] - zref) * a.c, p = exp2_fast(lz);
            s[1] += p;
            if (!(p <= 0.0f)) s[2] += p * lz;
            if (col < 0 || col >= a.ncols) s[5] = __int_as_float(0x7fffffff);
            if (j >= 0 && j < (int64_t)n * N && col >= 0 && col < a.ncols) {
                const float u = (to_float(elem[j]) - mx) * a.c;
                s[3] += p;
                if (!(p <= 0.0f)) s[4] += p * u;
                if (REST && (e == lo || a.crd[e - 1] != col)) s[5] += exp2_fast(u);
            }
        }
    }
    cta_reduce<6, DW, false>(s, room);
    cluster_wait();                                // the others are there
    if (tid < (int)ranks) {
        Told *to = &told[rank];
        store_peer(&to->m, tid, m[0]);
        store_peer(&to->others, tid, s[0]);
        store_peer(&to->stored, tid, s[5]);
        store_peer(&to->p, tid, s[3]);
        store_peer(&to->pu, tid, s[4]);
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();

    float top = MINUS_INF, others = 0.0f, stored = 0.0f, pu = 0.0f;
    for (unsigned r = 0; r < ranks; r++) top = max_nan(top, told[r].m);
    if (top == MINUS_INF) top = 0.0f;
    for (unsigned r = 0; r < ranks; r++) {
        const Told &o = told[r];
        const float d = ((o.m == MINUS_INF ? 0.0f : o.m) - top) * a.c, f = exp2_fast(d);
        if (o.others != 0.0f) others += o.others * f;
        if (o.stored != 0.0f) stored += o.stored * f;
        if (o.p != 0.0f) pu += o.pu + o.p * d;
    }
    const float total = others + stored, l2 = total == 0.0f ? 0.0f : log2f(total);     // 0: every logit is -inf, and so is q's log
    const float left = REST ? fmaxf(0.0f, 1.0f - s[1]) : 0.0f, inv = REST ? 1.0f : 1.0f / s[1];
    const float by = w * a.by;
    T *g = GRAD ? (T *)a.grad + t * a.ldg : nullptr;
    if (GRAD) {
        const float of = counts ? (left > 0.0f && others > 0.0f ? by * (1.0f - left * (total / others)) : by) : 0.0f;
        const bool whole = (((uintptr_t)g ^ (uintptr_t)x) & 15) == 0;
        uint4 *to = (uint4 *)((uintptr_t)g & ~(uintptr_t)15) + first;
        if (whole) {
            for (int i = tid; i < n; i += DT) {
                Granule<T> o;
                float v[N];
                if (counts) {
                    ((const Granule<T> *)(part + i))->unpack(v);
#pragma unroll
                    for (int k = 0; k < N; k++) v[k] = of * exp2_fast(fmaf(v[k] - top, a.c, -l2));
                } else {
#pragma unroll
                    for (int k = 0; k < N; k++) v[k] = 0.0f;
                }
                const int col = col0 + i * N;
                if (col >= 0 && col + N <= a.ncols) {
                    o.pack(v);
                    to[i] = o.w;
                } else {
#pragma unroll
                    for (int k = 0; k < N; k++)
                        if (col + k >= 0 && col + k < a.ncols) g[col + k] = from_float<T>(v[k]);
                }
            }
        } else {
            for (int i = tid; i < n * N; i += DT)
                if (col0 + i >= 0 && col0 + i < a.ncols)
                    g[col0 + i] = from_float<T>(counts ? of * exp2_fast(fmaf(to_float(elem[i]) - top, a.c, -l2)) : 0.0f);
        }
        __syncthreads();
        if (counts) {
            const float zref = REST ? a.lse[t] * LOG2E : m[1];
            for (int64_t e = lo + tid; e < hi; e += DT) {
                const int64_t col = a.crd[e], j = col - col0;
                if (j < 0 || j >= (int64_t)n * N || col < 0 || col >= a.ncols || (e > lo && a.crd[e - 1] == col)) continue;
                float p = 0.0f;                    // repeated columns are next to each other: their sum
                for (int64_t f = e; f < hi && a.crd[f] == col; f++)
                    p += exp2_fast(REST ? fmaf((float)z[f], a.c, -zref) : ((float)z[f] - zref) * a.c);
                g[col] = from_float<T>(by * (exp2_fast(fmaf(to_float(elem[j]) - top, a.c, -l2)) - p * inv));
            }
        }
    }
    if (rank != 0) return;
    if (tid == 0) {
        float loss = 0.0f;
        if (counts) {
            if (REST)
                loss = s[2] - pu + s[1] * l2 + (left > 0.0f ? left * (log2f(left) - log2f(others) + l2) : 0.0f);
            else
                loss = (s[2] - pu) * inv - log2f(s[1]) + l2;
        }
        a.rows[t] = loss * LN2;
        last = last_of(a.counter, (unsigned)a.nrows);
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    __shared__ double sums[DW];
    double sum = 0.0;
    for (int64_t r = tid; r < a.nrows; r += DT) {
        const float wr = a.weight ? a.weight[r] : 1.0f;
        if (wr != 0.0f) sum += (double)wr * __ldcg(a.rows + r);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((tid & 31) == 0) sums[tid >> 5] = sum;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < DW; i++) sum += sums[i];
        *a.loss = (float)(sum * a.scale);
    }
}

template <typename T, typename TV, bool REST, bool GRAD>
static int launch_distill(DistillArgs a, cudaStream_t st)
{
    constexpr int N = Granule<T>::N;
    const int all = (a.ncols + 2 * N - 2) / N;     // granules of a row, wherever it starts
    int ranks = 1;
    while (ranks < MOST_CLUSTER && (ceil_div(all, ranks) * 16 > 32 * 1024 || (a.nrows * ranks < sm_count() * 2 && all / ranks >= 512))) ranks *= 2;
    a.slice = ((int)ceil_div(all, ranks) + 1) & ~1;
    const size_t smem = (size_t)a.slice * 16 + (REST ? ((size_t)a.slice * N + 127) / 128 * 16 : 0);
    if (a.slice * 16 > MOST_SLICE) return fail("distill_loss: rows of %d columns do not fit the shared memory of eight SMs", a.ncols);
    return launch_cluster(distill_kernel<T, TV, REST, GRAD>, (unsigned)(a.nrows * ranks), ranks, DT, smem, st, a);
}

template <typename T, typename TV>
static int launch_distill(const DistillArgs &a, cudaStream_t st)
{
    if (a.lse) return a.grad ? launch_distill<T, TV, true, true>(a, st) : launch_distill<T, TV, true, false>(a, st);
    return a.grad ? launch_distill<T, TV, false, true>(a, st) : launch_distill<T, TV, false, false>(a, st);
}

template <typename T>
static int distill_loss(int64_t nrows, int64_t ncols, const int64_t *pos, const int64_t *crd, const void *val, int32_t val_bytes, const float *lse,
                        const float *weight, const void *x, int64_t ldx, void *grad, int64_t ldg, const double *temperature_scale, float *rows,
                        float *loss, void *stream)
{
    clear_error();
    cudaStream_t st = (cudaStream_t)stream;
    const double temperature = temperature_scale[0], scale = temperature_scale[1];
    if (nrows < 0 || ncols <= 0) return fail("distill_loss: %lld rows of %lld columns", (long long)nrows, (long long)ncols);
    if (ldx < ncols || (grad && ldg < ncols)) return fail("distill_loss: leading dimension smaller than the number of columns");
    if (!(temperature > 0.0) || temperature > 1e30) return fail("distill_loss: temperature %g is not a positive number", temperature);
    if (val_bytes != 4 && val_bytes != 8) return fail("distill_loss: the teacher's values have 4 or 8 bytes");
    if (ncols > (int64_t)MOST_CLUSTER * MOST_SLICE / (int64_t)sizeof(T) - 64)
        return fail("distill_loss: rows of %lld columns do not fit the shared memory of eight SMs", (long long)ncols);
    if (nrows > 0x7fffffffLL / MOST_CLUSTER) return fail("distill_loss: more than 2^28 rows");
    if ((uintptr_t)x % sizeof(T) || (uintptr_t)grad % sizeof(T)) return fail("distill_loss: an address that is not a multiple of the element's size");
    if (nrows == 0) {
        CB_CUDA(cudaMemsetAsync(loss, 0, sizeof(float), st));
        return 0;
    }
    DistillArgs a = {nrows, (int)ncols, 0, pos, crd, val, lse, weight, x, ldx, grad, ldg, (float)((double)LOG2E_D / temperature),
                     (float)(scale / temperature), (float)scale, rows, loss, next_counter()};
    if (!a.counter) return 1;
    return val_bytes == 4 ? launch_distill<T, float>(a, st) : launch_distill<T, double>(a, st);
}

}  // namespace cb200

#define DISTILL(suffix, T)                                                                                                              \
    extern "C" int32_t comet_b200_dev_distill_loss_##suffix##_i64(                                                                       \
        int64_t nrows, int64_t ncols, const int64_t *pos, const int64_t *crd, const void *val, int32_t val_bytes, const float *lse,      \
        const float *weight, const void *x, int64_t ldx, void *grad, int64_t ldg, const double *temperature_scale, float *rows,          \
        float *loss, void *stream)                                                                                                       \
    {                                                                                                                                    \
        return cb200::distill_loss<T>(nrows, ncols, pos, crd, val, val_bytes, lse, weight, x, ldx, grad, ldg, temperature_scale, rows,   \
                                      loss, stream);                                                                                     \
    }
DISTILL(bf16, __nv_bfloat16)
DISTILL(f16, __half)
DISTILL(f32, float)
