// Distillation from a teacher's top logits: the teacher is a CSR matrix S (rows tokens, columns the vocabulary) of the logits
// it has listed, the student a dense matrix X.  With c = log2(e) / temperature, q = softmax(X / temperature) and
//   p_j = exp(z_j / temperature) / sum over the row's entries                      (without lse)
//   p_j = exp(z_j / temperature - lse), left = max(0, 1 - sum p)                   (with lse: the rest is one outcome)
// a row's loss is sum p (log p - log q) [+ left (log left - log q_rest), q_rest = the sum of q where nothing is stored], and
//   d loss / d x_j = (M q_j - p_j) / temperature where an entry is stored, q_j (M - left / q_rest) / temperature elsewhere,
// with M = sum p + left: 1, unless the list's probabilities exceed 1 and nothing is left.
// q_rest is a sum of its own, not 1 minus the rest: where the teacher lists nearly all, the difference would have no digits left.
//
// A cluster of CTAs takes a row: each has its part of the row copied into shared memory (16 bytes a copy, no registers), so
// X is read from HBM once, and the maximum, the sums and the gradient are three passes over shared memory.  What the CTAs of
// a row have to tell each other are five floats, written into each other's shared memory.
//
// Bound: HBM, the bytes of X and of the gradient, but the clock first: 4096 x 131072 bf16 with gradient take 487 us (4.42 TB/s) where the bytes take
// 328: 20 warps on an SM issue an instruction every second clock (dependences, the exponential unit 53 % of the time, the barriers of a
// row), and under this load the SM clock falls to about 1.5 GHz.  65536 columns of f16 without a gradient: 124 us, 72 by the bytes.
// Slices of 32 KB by 128 threads leave room for six CTAs on an SM, which fill each other's waits: 506 us at the time, with 64 KB and 256
// threads 514, with 32 KB and 256 threads 543.  A cluster that stays and goes from row to row, with the next one on its way: 495 to 640.
#include "logits.cuh"
#include "stream.cuh"

namespace cb200 {

static const int DT = 128, DW = DT / 32;
static const int SLICE = 48 * 1024;                // bytes of a row that a CTA gets if eight of them can take the row at that
static const int MOST_SLICE = 192 * 1024;          // and at most

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
    double inv;                  // 1 / temperature
    float c, by, scale;          // log2(e) / temperature, scale / temperature
    float *rows, *loss;
    unsigned *counter;           // null: another kernel adds the rows up
};

// log p and p of an entry.  With lse p is not normalised afterwards, and what it is off by is the rest's error too, so the difference
// that the exponential is taken of is rounded twice, its residue a factor of p: f32 products of the size of lse would leave p 1e-6 of
// itself off.  A row has tens of entries, whose f64 operations take no time that shows.  Without lse the difference is to the largest entry,
// in the entries' type: f32 ones lose nothing that their sum does not divide out (4096 x 65536 f16 without gradient: 124 us, 127 in f64).
struct Weight {
    float log, p;
};
__device__ __forceinline__ Weight weight_of(float log2)
{
    return {log2 * LN2, exp2_fast(log2)};
}
__device__ __forceinline__ Weight weight_of(double log)
{
    Weight w;
    w.log = (float)log;
    w.p = expf(w.log);
    if (w.log > -104.0f && w.log < 89.0f) w.p = fmaf(w.p, (float)(log - w.log), w.p);              // neither 0 nor infinite
    return w;
}

// What 1 - sum p may be by rounding alone, where lse is a sum of the entries' own: lse comes with some roundings of the size of lse and of the
// largest logit, 2^-22 of them together, exponentials and sums of up to 32 numbers a thread add 2^-19.  A rest within it counts as none where
// no column is left for it, instead of making the loss infinite.
__device__ __forceinline__ float rounding_of(float lse, float most) { return fminf(0x1p-20f * (2.0f + fabsf(lse) + fabsf(most)), 0.5f); }

// what a CTA tells the others of its row: the maximum of its part, sums of 2^((x - maximum) c) of elements that are not
// stored and of those that are, of p's weights and of p's weights times (x - maximum) c
struct Told {
    float m, others, stored, p, pu;
};

// (x - m) c.  Where m c is less than NEAR it is x c - m c, one operation, and the rounding of m c is a factor that all of a CTA's
// terms and their sum have alike; `lacks` is what it is off by, which a CTA on the other side of NEAR has to know.
struct Exponent {
    float c, m, mc, lacks;
    bool near;
    __device__ __forceinline__ Exponent(float most, float c_) : c(c_), m(most == MINUS_INF ? 0.0f : most)
    {
        mc = m * c;
        near = fabsf(mc) < NEAR;
        lacks = near ? fmaf(m, c, -mc) : 0.0f;
    }
    __device__ __forceinline__ float of(float x) const { return near ? fmaf(x, c, -mc) : (x - m) * c; }
    __device__ __forceinline__ float2 of(float2 x) const { return fma2(x, make_float2(c, c), make_float2(-mc, -mc)); }      // near
    __device__ __forceinline__ float to(const Exponent &o) const { return near && o.near ? mc - o.mc : (m - o.m) * c - lacks + o.lacks; }
};

template <int N>
__device__ __forceinline__ float sum_of(const float (&v)[N])
{
    float s = v[0];
#pragma unroll
    for (int i = 1; i < N; i++) s += v[i];
    return s;
}

// scale * the sum of weight * rows, by one warp or more, in a fixed order; the result in thread 0
template <int THREADS>
__device__ __forceinline__ void add_rows(const DistillArgs &a, double *room)
{
    double sum = 0.0;
    for (int64_t r = threadIdx.x; r < a.nrows; r += THREADS) {
        const float w = a.weight ? a.weight[r] : 1.0f;
        if (w != 0.0f) sum += (double)w * __ldcg(a.rows + r);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (THREADS > 32) {
        if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = sum;
        __syncthreads();
        if (threadIdx.x == 0)
            for (int i = 1; i < THREADS / 32; i++) sum += room[i];
    }
    if (threadIdx.x == 0) *a.loss = (float)(sum * a.scale);
}

__global__ void __launch_bounds__(1024)
distill_sum_kernel(const DistillArgs a)
{
    __shared__ double room[32];
    wait_for_previous();
    add_rows<1024>(a, room);
}

template <typename T, typename TV, bool REST, bool GRAD>
__global__ void __launch_bounds__(DT)
distill_kernel(const DistillArgs a)
{
    constexpr int N = Granule<T>::N;
    extern __shared__ uint4 dyn[];
    __shared__ float most[DW], sums[6][DW];
    __shared__ TV zmost[DW];
    __shared__ Told told[MOST_CLUSTER];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned rank = cluster_rank(), ranks = cluster_size();
    const int64_t t = blockIdx.x / ranks, lo = a.pos[t], hi = a.pos[t + 1];
    const float w = a.weight ? a.weight[t] : 1.0f;
    const T *x = (const T *)a.x + t * a.ldx;
    T *g = GRAD ? (T *)a.grad + t * a.ldg : nullptr;
    const TV *z = (const TV *)a.val;
    // the row's granules, and this CTA's; element e of them is column e - off + first * N
    const int off = (int)((uintptr_t)x & 15) / (int)sizeof(T);
    const int all = (off + a.ncols + N - 1) / N, first = min((int)rank * a.slice, all), n = min(a.slice, all - first);
    const int col0 = first * N - off;              // the column of this CTA's element 0; negative if that lies before the row
    Granule<T> *part = (Granule<T> *)dyn;
    uint32_t *bits = (uint32_t *)(dyn + a.slice);  // a bit per element: stored
    T *elem = (T *)dyn;
    const bool entries = lo + warp * 32 < hi;      // the warp has some of the row's

    TV zm = MINUS_INF;
    if (lo < hi && w != 0.0f) {
        if (ranks > 1) cluster_arrive_relaxed();   // only to say that it is there
        const uint4 *from = (const uint4 *)((uintptr_t)x & ~(uintptr_t)15) + first;
        {
            const uint32_t to = (uint32_t)__cvta_generic_to_shared(part);
            int i = tid;
            for (; i + 3 * DT < n; i += 4 * DT) {
                copy_far<0>(to + i * 16, from + i);
                copy_far<DT * 16>(to + i * 16, from + i);
                copy_far<DT * 32>(to + i * 16, from + i);
                copy_far<DT * 48>(to + i * 16, from + i);
            }
            for (; i < n; i += DT) copy_far<0>(to + i * 16, from + i);
        }
        if (REST)
            for (int i = tid; i < (n * N + 31) / 32; i += DT) bits[i] = 0;
        for (int64_t e = lo + tid; e < hi; e += DT) zm = max_nan(zm, z[e]);
        if (entries) zm = warp_max(zm);
        wait_copies();
        float m = MINUS_INF;
        if (tid < n) {
#pragma unroll
            for (int side = 0; side < 2; side++) { // elements before and behind the row
                const int i = side ? n - 1 : 0;
                if (tid == i % DT && (col0 + i * N < 0 || col0 + i * N + N > a.ncols))
                    for (int k = 0; k < N; k++)
                        if (col0 + i * N + k < 0 || col0 + i * N + k >= a.ncols) elem[i * N + k] = from_float<T>(MINUS_INF);
            }
            typename Granule<T>::Most mm = part[tid].most();
#pragma unroll 4
            for (int i = tid + DT; i < n; i += DT) mm = most_of(mm, part[i].most());
            m = to_float(largest(mm));
        }
        m = warp_max(m);
        if (lane == 0) {
            most[warp] = m;
            zmost[warp] = entries ? zm : (TV)MINUS_INF;
        }
        __syncthreads();
        zm = zmost[0];
#pragma unroll
        for (int i = 1; i < DW; i++) zm = max_nan(zm, zmost[i]);
    }
    if (zm == MINUS_INF) {                         // the row does not count
        if (GRAD) {
            uint4 *to = (uint4 *)((uintptr_t)g & ~(uintptr_t)15) + first;
            const bool alike = (((uintptr_t)g ^ (uintptr_t)x) & 15) == 0;
            for (int i = tid; i < n; i += DT) {
                const int col = col0 + i * N;
                if (alike && col >= 0 && col + N <= a.ncols) {
                    to[i] = make_uint4(0, 0, 0, 0);
                } else {
                    for (int k = 0; k < N; k++)
                        if (col + k >= 0 && col + k < a.ncols) g[col + k] = from_float<T>(0.0f);
                }
            }
        }
        __syncwarp();
        if (lo < hi && w != 0.0f && ranks > 1) cluster_wait();
        if (rank != 0 || warp != 0) return;
        if (lane == 0) a.rows[t] = 0.0f;
    } else {
        float m = most[0];
#pragma unroll
        for (int i = 1; i < DW; i++) m = max_nan(m, most[i]);
        const Exponent u(m, a.c);
        if (REST) {
            for (int64_t e = lo + tid; e < hi; e += DT) {
                const int64_t j = a.crd[e] - col0;
                if (j >= 0 && j < (int64_t)n * N) atomicOr(&bits[j >> 5], 1u << (j & 31));
            }
            __syncthreads();
        }
        float2 s2 = make_float2(0.0f, 0.0f);
        if (u.near) {
#pragma unroll 4
            for (int i = tid; i < n; i += DT) {
                float2 v[N / 2];
                part[i].unpack(v);
#pragma unroll
                for (int k = 0; k < N / 2; k++) {
                    v[k] = u.of(v[k]);
                    v[k] = make_float2(exp2_fast(v[k].x), exp2_fast(v[k].y));
                }
                if (REST) {
                    const unsigned skip = N == 8 ? ((const uint8_t *)bits)[i] : ((const uint8_t *)bits)[i >> 1] >> ((i & 1) * 4) & 15;
                    if (skip)
#pragma unroll
                        for (int k = 0; k < N / 2; k++) {
                            if (skip >> (2 * k) & 1) v[k].x = 0.0f;
                            if (skip >> (2 * k + 1) & 1) v[k].y = 0.0f;
                        }
                }
#pragma unroll
                for (int k = 0; k < N / 2; k++) s2 = add2(s2, v[k]);
            }
        } else {
            for (int i = tid; i < n * N; i += DT)
                if (!REST || !(bits[i >> 5] >> (i & 31) & 1)) s2.x += exp2_fast(u.of(to_float(elem[i])));
        }
        s2.x = warp_sum(s2.x + s2.y);
        // of the entries: p's weights, times their logarithm; in this part: weights, times (x - m) c, and stored columns' 2^((x - m) c)
        float s[5] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        const double sum = REST ? a.lse[t] : 0.0;
        auto weight = [&](int64_t e) {
            if constexpr (REST) return weight_of(fma((double)z[e], a.inv, -sum));
            else if constexpr (sizeof(TV) == 8) return weight_of((z[e] - zm) * a.inv);
            else return weight_of((z[e] - zm) * a.c);
        };
        if (entries) {
            for (int64_t e = lo + tid; e < hi; e += DT) {
                const int64_t col = a.crd[e], j = col - col0;
                const Weight y = weight(e);
                const float p = y.p;
                s[0] += p;
                if (!(p <= 0.0f)) s[1] += p * y.log;
                if (col < 0 || col >= a.ncols) {
                    s[1] = __int_as_float(0x7fffffff);
                } else if (j >= 0 && j < (int64_t)n * N) {
                    const float v = u.of(to_float(elem[j]));
                    s[2] += p;
                    if (!(p <= 0.0f)) s[3] += p * v;
                    if (REST && (e == lo || a.crd[e - 1] != col)) s[4] += exp2_fast(v);
                }
            }
#pragma unroll
            for (int i = 0; i < 5; i++) s[i] = warp_sum(s[i]);
        }
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < 5; i++) sums[i][warp] = s[i];
            sums[5][warp] = s2.x;
        }
        __syncthreads();
        if (ranks > 1) cluster_wait();             // the others are there
        if (warp == 0 && lane < (int)ranks) {
            const float others = sum_of(sums[5]), stored = sum_of(sums[4]), p = sum_of(sums[2]), pu = sum_of(sums[3]);
            if (ranks > 1) {
                Told *to = &told[rank];
                store_peer(&to->m, lane, m);
                store_peer(&to->others, lane, others);
                store_peer(&to->stored, lane, stored);
                store_peer(&to->p, lane, p);
                store_peer(&to->pu, lane, pu);
            } else {
                told[0] = {m, others, stored, p, pu};
            }
        }
        if (ranks > 1) {
            __syncwarp();
            cluster_arrive();
            cluster_wait();
        } else {
            __syncthreads();
        }
        if (!GRAD && (rank != 0 || warp != 0)) return;
        // the row's: a lane per CTA
        const Told &o = told[lane & (MOST_CLUSTER - 1)];
        const bool there = (lane & (MOST_CLUSTER - 1)) < (int)ranks;
        const Exponent top(warp_max(there ? o.m : MINUS_INF), a.c);
        const float d = there ? Exponent(o.m, a.c).to(top) : 0.0f, f = exp2_fast(d);
        float others = there && o.others != 0.0f ? o.others * f : 0.0f, stored = there && o.stored != 0.0f ? o.stored * f : 0.0f;
        float pu = there && o.p != 0.0f ? o.pu + o.p * d : 0.0f;
#pragma unroll
        for (int i = 1; i < MOST_CLUSTER; i *= 2) {
            others += __shfl_xor_sync(0xffffffffu, others, i);
            stored += __shfl_xor_sync(0xffffffffu, stored, i);
            pu += __shfl_xor_sync(0xffffffffu, pu, i);
        }
        const float total = REST ? others + stored : others, p = sum_of(sums[0]);
        float left = REST ? fmaxf(0.0f, 1.0f - p) : 0.0f;
        if (REST && others == 0.0f && left <= rounding_of((float)sum, (float)(zm * a.inv))) left = 0.0f;
        if (GRAD) {
            const float by = w * a.by, sum_p = REST && left == 0.0f ? p : 1.0f;
            const float part_of = total == 0.0f ? 0.0f : sum_p * __fdividef(by, total);             // total 0: every logit is -inf
            const float of = left > 0.0f && others > 0.0f ? part_of * (1.0f - left * (total / others)) : part_of;
            const bool alike = (((uintptr_t)g ^ (uintptr_t)x) & 15) == 0;
            if (alike && top.near && col0 >= 0 && col0 + n * N <= a.ncols) {            // no granule that is not all the row's
                uint4 *to = (uint4 *)((uintptr_t)g & ~(uintptr_t)15) + first;
                const float2 of2 = make_float2(of, of);
#pragma unroll 4
                for (int i = tid; i < n; i += DT) {
                    float2 v[N / 2];
                    part[i].unpack(v);
#pragma unroll
                    for (int k = 0; k < N / 2; k++) {
                        v[k] = top.of(v[k]);
                        v[k] = mul2(make_float2(exp2_fast(v[k].x), exp2_fast(v[k].y)), of2);
                    }
                    Granule<T> out;
                    out.pack(v);
                    to[i] = out.w;
                }
            } else if (alike && top.near) {
                uint4 *to = (uint4 *)((uintptr_t)g & ~(uintptr_t)15) + first;
#pragma unroll 4
                for (int i = tid; i < n; i += DT) {
                    float2 v[N / 2];
                    part[i].unpack(v);
#pragma unroll
                    for (int k = 0; k < N / 2; k++) {
                        v[k] = top.of(v[k]);
                        v[k] = mul2(make_float2(exp2_fast(v[k].x), exp2_fast(v[k].y)), make_float2(of, of));
                    }
                    Granule<T> out;
                    out.pack(v);
                    const int col = col0 + i * N;
                    if (col >= 0 && col + N <= a.ncols) {
                        to[i] = out.w;
                    } else {
                        for (int k = 0; k < N; k++)
                            if (col + k >= 0 && col + k < a.ncols) g[col + k] = ((const T *)&out)[k];
                    }
                }
            } else {
                for (int i = tid; i < n * N; i += DT)
                    if (col0 + i >= 0 && col0 + i < a.ncols) g[col0 + i] = from_float<T>(of * exp2_fast(top.of(to_float(elem[i]))));
            }
            __syncthreads();
            const float inv = REST ? 1.0f : __fdividef(1.0f, p);
            for (int64_t e = lo + tid; e < hi; e += DT) {
                const int64_t col = a.crd[e], j = col - col0;
                if (j < 0 || j >= (int64_t)n * N || col < 0 || col >= a.ncols || (e > lo && a.crd[e - 1] == col)) continue;
                float pj = 0.0f;                   // repeated columns are next to each other: their sum
                for (int64_t i = e; i < hi && a.crd[i] == col; i++) pj += weight(i).p;
                g[col] = from_float<T>(part_of * exp2_fast(top.of(to_float(elem[j]))) - by * (pj * inv));
            }
            if (rank != 0 || warp != 0) return;
        }
        const float l2 = total == 0.0f ? 0.0f : log2f(total), plogp = sum_of(sums[1]);
        if (lane == 0) {
            a.rows[t] = REST ? fmaf(p * l2 - pu + (left > 0.0f ? left * (log2f(left) - log2f(others) + l2) : 0.0f), LN2, plogp)
                             : (plogp - pu * LN2) / p + (l2 - log2f(p)) * LN2;
        }
    }
    if (!a.counter) return;
    unsigned last = 0;
    if (lane == 0) last = last_of(a.counter, (unsigned)a.nrows);
    if (!__shfl_sync(0xffffffffu, last, 0)) return;
    __threadfence();
    add_rows<32>(a, nullptr);
}

template <typename T, typename TV, bool REST, bool GRAD>
static int launch_distill(DistillArgs a, cudaStream_t st)
{
    constexpr int N = Granule<T>::N;
    const int all = (a.ncols + 2 * N - 2) / N;     // granules of a row, wherever it starts
    int ranks = 1;
    while (ranks < MOST_CLUSTER && (ceil_div(all, ranks) * 16 > SLICE + 64 || (a.nrows * ranks < sm_count() && all / ranks >= 2 * DT))) ranks *= 2;
    a.slice = ((int)ceil_div(all, ranks) + 1) & ~1;
    auto room = [](size_t granules) { return granules * 16 + (REST ? (granules * N + 127) / 128 * 16 : 0); };
    if (a.slice * 16 > MOST_SLICE) return fail("distill_loss: rows of %d columns do not fit the shared memory of eight SMs", a.ncols);
    const bool few = a.nrows <= 256;               // the last row's warp adds them up
    if (!few) a.counter = nullptr;
    CB_TRY(launch_cluster(distill_kernel<T, TV, REST, GRAD>, (unsigned)(a.nrows * ranks), ranks, DT, room(a.slice), room(MOST_SLICE / 16), st, a));
    if (!few) CB_CUDA(launch_behind(distill_sum_kernel, dim3(1), 1024, 0, st, a));
    return 0;
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
    if (!temperature_fits(temperature)) return fail("distill_loss: temperature %g is not a number of 1e-38 to 1e30", temperature);
    if (val_bytes != 4 && val_bytes != 8) return fail("distill_loss: the teacher's values have 4 or 8 bytes");
    if (ncols > (int64_t)MOST_CLUSTER * MOST_SLICE / (int64_t)sizeof(T) - 64)
        return fail("distill_loss: rows of %lld columns do not fit the shared memory of eight SMs", (long long)ncols);
    if (nrows > 0x7fffffffLL / MOST_CLUSTER) return fail("distill_loss: more than 2^28 rows");
    if ((uintptr_t)x % sizeof(T) || (uintptr_t)grad % sizeof(T)) return fail("distill_loss: an address that is not a multiple of the element's size");
    if (nrows == 0) {
        CB_CUDA(cudaMemsetAsync(loss, 0, sizeof(float), st));
        return 0;
    }
    DistillArgs a = {nrows, (int)ncols, 0, pos, crd, val, lse, weight, x, ldx, grad, ldg, 1.0 / temperature, (float)((double)LOG2E_D / temperature),
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
