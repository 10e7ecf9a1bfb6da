// The balance loss of a router: S (CSR, rows tokens, columns experts) says which experts took which tokens, R are the router's
// logits.  A row is active if it stores something and its mask is not 0.  With N active rows and K entries in a sequence,
// f_e = (entries in column e) / K and P_e = the mean over active rows of p_e, p = softmax(R) or sigmoid(R) / sum sigmoid(R):
//   loss = scale * (mean over sequences with active rows of  E * sum_e f_e P_e)
//   d loss / d r_e = scale E / (sequences N) * p_e (f_e - sum_j f_j p_j)          [times (1 - sigmoid(r_e))]
// The counts are all that the gradient needs of other rows, so they come first and R is read once.  f is used as
// g = f - 1 / E, taken from whole numbers: for balanced experts the difference f_e - sum f p would lose its digits otherwise.
// Where every sigmoid of a row underflows, their shares are those of e^(r - max) / (1 + e^r).
//
// Small batches: one cluster counts, exchanges its counts through shared memory and takes the rows, in one launch.  Otherwise a
// kernel counts and a second one, whose start overlaps with it, takes the rows.
// A group of lanes takes a row, 16 bytes a lane or a few times that: a lane's columns are the same in every row, so their g stay in
// registers while the sequence lasts.
//
// Bound: HBM, R and its gradient; small batches: the launch.  65536 x 256 bf16 in 32 sequences, sigmoid: 40 us, 11 by the bytes; counting 5, rows 34,
// which are 276 instructions a row.  16384 x 64 f32: 16.6 us, most of it the two launches and their chains of loads.  128 x 8: 4.6 us on
// the device, 14 a call.  With the counters cleared by the driver and a warp per row whatever its length: 155, 47 and 23.
#include "logits.cuh"
#include "stream.cuh"

namespace cb200 {

static const int BT = 256, BW = BT / 32, MOST_EXPERTS = 1024;
// Logits of the one-launch kernel.  bf16, one launch against two, us on the device (calls in a graph): 128 rows of 64 6.3, 8.1; 1000 of 64 7.9, 8.1; 250 of 256 8.2,
// 8.6; 63 of 1024 9.6, 11.3; 4096 of 8 7.4, 8.0, but 8000 of 8 10.8, 8.1.  2048 rows of 64 would take 2 us more than with two.  The host spends a launch less, too.
static const int64_t SMALL_ELEMENTS = 65536;
static const int SMALL_COUNTS = 2048;              // sequences times (experts + 2) that the one-launch kernel holds
static const int KEPT_COUNTS = 16384;              // and that are counted in memory that every call leaves at 0

typedef unsigned long long u64;
static __device__ u64 g_kept[KEPT_COUNTS + 2];

// What the counting leaves: counts[sequence][expert], and {active rows, entries} per sequence; in `all`: sequences with active rows, and
// whether a column was outside.
struct Tally {
    u64 *counts, *rows, *all;
};

struct BalanceArgs {
    int64_t nrows;
    int ncols;
    const int64_t *pos, *crd;
    int64_t nseq;
    const int64_t *seq;
    const uint8_t *mask;
    const void *r;
    int64_t ldr;
    void *grad;
    int64_t ldg;
    float scale;
    bool whole;                  // rows of R and of the gradient begin at 16 bytes and are a whole number of them
    Tally tally;
    bool kept;                   // the tally is g_kept
    int64_t *counts;
    double *partial;
    float *loss;
    unsigned *counter;
};

__device__ __forceinline__ int64_t sequence_of(const int64_t *seq, int64_t nseq, int64_t row)
{
    int64_t lo = 0, hi = nseq - 1;                 // the last sequence that begins at or before the row
    while (lo < hi) {
        const int64_t mid = (lo + hi + 1) / 2;
        if (seq[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Counts rows [r0, r1) by one warp, 32 at a time: hit(sequence, column) for each entry of an active row, rows(sequence, active, entries)
// for sums over lanes of one sequence, by one lane.  Where all 32 rows store the same number, their entries are read side by side.
template <typename Hit, typename Rows, typename Bad>
__device__ __forceinline__ void count_rows(const BalanceArgs &a, int64_t r0, int64_t r1, Hit hit, Rows rows, Bad bad)
{
    const int lane = threadIdx.x & 31;
    for (int64_t b = r0; b < r1; b += 32) {
        const int64_t t = b + lane;
        int64_t lo = 0, hi = 0, s = 0;
        if (t < r1) {
            lo = a.pos[t];
            hi = a.pos[t + 1];
            if (a.seq) s = sequence_of(a.seq, a.nseq, t);
        }
        const bool active = hi > lo && (!a.mask || a.mask[t]);
        const unsigned on = __ballot_sync(0xffffffffu, active);
        if (!on) continue;
        const int64_t lo0 = __shfl_sync(0xffffffffu, (long long)lo, 0), s0 = __shfl_sync(0xffffffffu, (long long)s, __ffs(on) - 1);
        const int n = (int)min(hi - lo, (int64_t)0x7fffffff), n0 = __shfl_sync(0xffffffffu, n, 0);
        const bool one = __all_sync(0xffffffffu, s == s0 || !active);
        if (one && n0 > 0 && n0 <= 64 && __all_sync(0xffffffffu, t >= r1 || n == n0)) {
            const int many = 32 * n0;
            for (int i0 = lane; i0 < many; i0 += 32 * 8) {     // eight at a time on their way
                int64_t j[8];
                unsigned have = 0;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const int i = i0 + 32 * k;
                    if (i < many && on >> (i / n0) & 1) {
                        j[k] = a.crd[lo0 + i];
                        have |= 1u << k;
                    }
                }
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (have >> k & 1) {
                        if (j[k] >= 0 && j[k] < a.ncols) hit(s0, (int)j[k]);
                        else bad();
                    }
            }
        } else if (active) {
            for (int64_t e = lo; e < hi; e++) {
                const int64_t j = a.crd[e];
                if (j >= 0 && j < a.ncols) hit(s, (int)j);
                else bad();
            }
        }
        if (one) {
            int64_t sum = active ? hi - lo : 0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, (long long)sum, o);
            if (lane == 0) rows(s0, __popc(on), sum);
        } else if (active) {
            rows(s, 1, hi - lo);
        }
    }
}

// A row as a lane has it ahead of time.
template <int Q>
struct NextRow {
    uint4 x[Q];
    bool active;
};

// Rows [r0, r1) of a warp, G lanes and Q times 16 bytes a lane each; the next rows are on their way while these are computed.  WHOLE: every granule is
// 16 aligned bytes of one row.  Returns the lane's part of the loss.
template <typename T, int G, int Q, bool SIGMOID, bool WHOLE>
__device__ __forceinline__ double take_rows(const BalanceArgs &a, const Tally &tally, int64_t r0, int64_t r1)
{
    constexpr int N = Granule<T>::N, AT_ONCE = 32 / G;
    const int lane = threadIdx.x & 31, l = lane % G;
    const float sequences = (float)tally.all[0], share = 1.0f / (float)a.ncols;
    int64_t s_end = -1;                            // the row at which the lane's sequence ends
    float g[Q * N], by = 0.0f;
    double sum = 0.0;
    auto has = [&](int q, int e) { return (q * G + l) * N + e < a.ncols; };
    auto fetch = [&](int64_t t) {
        NextRow<Q> n;
        n.active = false;
        if (t < r1) {
            const T *r = (const T *)a.r + t * a.ldr;
#pragma unroll
            for (int q = 0; q < Q; q++) {
                if (WHOLE) {
                    if (has(q, 0)) n.x[q] = ((const uint4 *)r)[q * G + l];       // no read-only load: the gradient may be R
                } else {
                    T *v = (T *)&n.x[q];
#pragma unroll
                    for (int e = 0; e < N; e++) v[e] = has(q, e) ? r[(q * G + l) * N + e] : from_float<T>(MINUS_INF);
                }
            }
            n.active = a.pos[t] < a.pos[t + 1] && (!a.mask || a.mask[t]);
        }
        return n;
    };
    NextRow<Q> next = fetch(r0 + lane / G);
    for (int64_t b = r0; b < r1; b += AT_ONCE) {
        const int64_t t = b + lane / G;
        const bool there = t < r1;
        const NextRow<Q> now = next;
        next = fetch(t + AT_ONCE);
        const bool active = now.active;
        T *grad = a.grad ? (T *)a.grad + t * a.ldg : nullptr;
        if (!__any_sync(0xffffffffu, active)) {    // nothing but zeros
            if (grad && there)
#pragma unroll
                for (int q = 0; q < Q; q++) {
                    if (WHOLE) {
                        if (has(q, 0)) ((uint4 *)grad)[q * G + l] = make_uint4(0, 0, 0, 0);
                    } else {
#pragma unroll
                        for (int e = 0; e < N; e++)
                            if (has(q, e)) grad[(q * G + l) * N + e] = from_float<T>(0.0f);
                    }
                }
            continue;
        }
        if (there && t >= s_end) {
            int64_t s = 0;
            s_end = a.nrows;
            if (a.seq) {
                s = sequence_of(a.seq, a.nseq, t);
                if (s + 1 < a.nseq) s_end = a.seq[s + 1];
            }
            const int64_t entries = (int64_t)tally.rows[2 * s + 1];
            by = a.scale * (float)a.ncols / (sequences * (float)tally.rows[2 * s]);
            const float unit = (float)(1.0 / ((double)entries * a.ncols));
#pragma unroll
            for (int q = 0; q < Q; q++)
#pragma unroll
                for (int e = 0; e < N; e++)
                    g[q * N + e] = has(q, e) ? (float)((int64_t)tally.counts[s * a.ncols + (q * G + l) * N + e] * a.ncols - entries) * unit : 0.0f;
        }
        float v[Q * N], slope[SIGMOID ? Q * N : 1];
        // the lane's logits; -inf where there is no column
        auto logits = [&](float (&u)[Q * N]) {
#pragma unroll
            for (int q = 0; q < Q; q++) {
                Granule<T> x;
                x.w = now.x[q];
                if (WHOLE && !has(q, 0)) x = Granule<T>::least();
                float each[N];
                x.unpack(each);
#pragma unroll
                for (int e = 0; e < N; e++) u[q * N + e] = each[e];
            }
        };
        float p = 0.0f, gp = 0.0f;
        auto add_up = [&]() {
            p = gp = 0.0f;
#pragma unroll
            for (int i = 0; i < Q * N; i++) {
                p += v[i];
                gp = fmaf(v[i], g[i], gp);
            }
#pragma unroll
            for (int o = G / 2; o > 0; o >>= 1) {
                p += __shfl_xor_sync(0xffffffffu, p, o);
                gp += __shfl_xor_sync(0xffffffffu, gp, o);
            }
        };
        auto maximum = [&](const float (&u)[Q * N]) {
            float m = u[0];
#pragma unroll
            for (int i = 1; i < Q * N; i++) m = max_nan(m, u[i]);
            if (G == 32) m = warp_max(m);
            else
#pragma unroll
                for (int o = G / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
            return m == MINUS_INF ? 0.0f : m;      // exp(-inf - 0) = 0: a row of -inf has no scores
        };
        logits(v);
        if (SIGMOID) {
#pragma unroll
            for (int i = 0; i < Q * N; i++) {
                const float d = min_nan(exp2_fast(v[i] * -LOG2E), 1e38f);
                v[i] = reciprocal(1.0f + d);
                slope[i] = d * v[i];
            }
            add_up();
            if (__any_sync(0xffffffffu, active && p < 1e-30f)) {               // sigmoids below f32's range, or none: their shares by e^(r - max) / (1 + e^r)
                float low[Q * N];
                logits(low);
                const float m = fminf(maximum(low), 0.0f);
#pragma unroll
                for (int i = 0; i < Q * N; i++) {
                    slope[i] = reciprocal(1.0f + min_nan(exp2_fast(low[i] * LOG2E), 1e38f));
                    v[i] = low[i] > 60.0f ? exp2_fast(-m * LOG2E) : exp2_fast((low[i] - m) * LOG2E) * slope[i];
                }
                add_up();
            }
        } else {
            const float m = maximum(v);
#pragma unroll
            for (int i = 0; i < Q * N; i++) v[i] = exp2_fast((v[i] - m) * LOG2E);
            add_up();
        }
        const float inv = p == 0.0f ? 0.0f : reciprocal(p);
        gp *= inv;
        if (l == 0 && active && p != 0.0f) sum += (double)(by * (share + gp));
        if (grad && there) {
            const float f = by * inv;
#pragma unroll
            for (int i = 0; i < Q * N; i++) {
                v[i] = f * v[i] * (g[i] - gp);
                if (SIGMOID) v[i] *= slope[i];
                if (G < 32 && !active) v[i] = 0.0f;            // its logits may be anything
            }
#pragma unroll
            for (int q = 0; q < Q; q++) {
                float u[N];
#pragma unroll
                for (int e = 0; e < N; e++) u[e] = v[q * N + e];
                if (WHOLE) {
                    Granule<T> x;
                    x.pack(u);
                    if (has(q, 0)) ((uint4 *)grad)[q * G + l] = x.w;
                } else {
#pragma unroll
                    for (int e = 0; e < N; e++)
                        if (has(q, e)) grad[(q * G + l) * N + e] = from_float<T>(u[e]);
                }
            }
        }
    }
    return sum;
}

// The CTA's sum, in thread 0, in a fixed order.
__device__ __forceinline__ double cta_sum(double v, double *room)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int i = 1; i < BW; i++) v += room[i];
    return v;
}

// All of a small batch by one cluster.
template <typename T, int G, int Q, bool SIGMOID, bool WHOLE>
__global__ void __launch_bounds__(BT)
balance_small_kernel(const BalanceArgs a)
{
    __shared__ int hits[SMALL_COUNTS + 1];         // counts, {rows, entries} per sequence, a column outside
    __shared__ u64 total[SMALL_COUNTS + 2];
    __shared__ double room[BW], parts[MOST_CLUSTER];
    const int tid = threadIdx.x, many = (int)a.nseq * a.ncols, words = many + 2 * (int)a.nseq + 1;
    const unsigned rank = cluster_rank(), ranks = cluster_size();
    for (int i = tid; i < words; i += BT) hits[i] = 0;
    if (tid == 0) total[words] = 0;
    __syncthreads();
    const int64_t warps = (int64_t)ranks * BW, w = (int64_t)rank * BW + (tid >> 5);
    const int64_t per = (a.nrows + warps * 32 - 1) / (warps * 32) * 32, r0 = min(w * per, a.nrows), r1 = min(r0 + per, a.nrows);
    count_rows(a, r0, r1, [&](int64_t s, int j) { atomicAdd(&hits[(int)s * a.ncols + j], 1); },
               [&](int64_t s, int n, int64_t e) {
                   atomicAdd(&hits[many + 2 * (int)s], n);
                   atomicAdd(&hits[many + 2 * (int)s + 1], (int)e);
               },
               [&]() { hits[words - 1] = 1; });
    if (ranks > 1) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    } else {
        __syncthreads();
    }
    for (int i = tid; i < words; i += BT) {
        u64 n = 0;
        for (unsigned k = 0; k < ranks; k++) n += (u64)(ranks > 1 ? peer_load(&hits[i], k) : hits[i]);
        total[i] = n;
        if (rank == 0 && i < many) a.counts[i] = (int64_t)n;
        if (i >= many && i < words - 1 && (i - many) % 2 == 0 && n) atomicAdd(&total[words], 1ull);
    }
    __syncthreads();
    const Tally tally = {total, total + many, total + words};
    const int64_t each = (a.nrows + warps - 1) / warps, q0 = min(w * each, a.nrows), q1 = min(q0 + each, a.nrows);
    const double sum = cta_sum(take_rows<T, G, Q, SIGMOID, WHOLE>(a, tally, q0, q1), room);
    if (ranks > 1) {
        if (tid == 0) store_peer(&parts[rank], 0, sum);
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    } else if (tid == 0) {
        parts[0] = sum;
    }
    if (rank != 0 || tid != 0) return;
    double loss = 0.0;
    for (unsigned k = 0; k < ranks; k++) loss += parts[k];
    *a.loss = total[words - 1] ? __int_as_float(0x7fffffff) : (float)loss;
}

// Counts of a larger batch: a CTA's rows of one sequence in shared memory first.
__global__ void __launch_bounds__(BT)
balance_count_kernel(const BalanceArgs a, int64_t per)
{
    __shared__ int hits[MOST_EXPERTS];
    let_next_start();
    const int64_t c0 = (int64_t)blockIdx.x * per, c1 = min(c0 + per, a.nrows);
    const int64_t s0 = a.seq && c0 < a.nrows ? sequence_of(a.seq, a.nseq, c0) : 0;
    for (int i = threadIdx.x; i < a.ncols; i += BT) hits[i] = 0;
    __syncthreads();
    wait_for_previous();                           // the call before has left the tally at 0
    const int64_t each = (per / BW + 31) / 32 * 32, r0 = min(c0 + (threadIdx.x >> 5) * each, c1), r1 = min(r0 + each, c1);
    const Tally &y = a.tally;
    count_rows(a, r0, r1,
               [&](int64_t s, int j) {
                   if (s == s0) atomicAdd(&hits[j], 1);
                   else atomicAdd(&y.counts[s * a.ncols + j], 1ull);
               },
               [&](int64_t s, int n, int64_t e) {
                   if (atomicAdd(&y.rows[2 * s], (u64)n) == 0) atomicAdd(&y.all[0], 1ull);
                   atomicAdd(&y.rows[2 * s + 1], (u64)e);
               },
               [&]() { y.all[1] = 1; });
    __syncthreads();
    for (int i = threadIdx.x; i < a.ncols; i += BT)
        if (hits[i]) atomicAdd(&y.counts[s0 * a.ncols + i], (u64)hits[i]);
}

// CTAs on an SM: as many as a lane's values leave registers for
template <typename T, int Q>
constexpr int balance_ctas() { return Q * Granule<T>::N <= 8 ? 4 : Q * Granule<T>::N <= 16 ? 2 : 1; }

template <typename T, int G, int Q, bool SIGMOID, bool WHOLE>
__global__ void __launch_bounds__(BT, balance_ctas<T, Q>())
balance_kernel(const BalanceArgs a)
{
    __shared__ double room[BW];
    __shared__ bool last;
    const int tid = threadIdx.x;
    const int64_t warps = (int64_t)gridDim.x * BW, w = (int64_t)blockIdx.x * BW + (tid >> 5);
    const int64_t each = (a.nrows + warps - 1) / warps, r0 = min(w * each, a.nrows), r1 = min(r0 + each, a.nrows);
    wait_for_previous();
    const int64_t many = a.nseq * a.ncols;
    if (a.kept)
        for (int64_t i = (int64_t)blockIdx.x * BT + tid; i < many; i += (int64_t)gridDim.x * BT) a.counts[i] = (int64_t)a.tally.counts[i];
    const double sum = cta_sum(take_rows<T, G, Q, SIGMOID, WHOLE>(a, a.tally, r0, r1), room);
    if (tid == 0) {
        a.partial[blockIdx.x] = sum;
        last = last_of(a.counter, gridDim.x);
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    double all = 0.0;
    for (int i = tid; i < (int)gridDim.x; i += BT) all += __ldcg(a.partial + i);
    all = cta_sum(all, room);
    if (tid == 0) *a.loss = a.tally.all[1] ? __int_as_float(0x7fffffff) : (float)all;
    if (a.kept) {
        __syncthreads();
        for (int i = tid; i < (int)many; i += BT) a.tally.counts[i] = 0;
        for (int i = tid; i < 2 * (int)a.nseq; i += BT) a.tally.rows[i] = 0;
        if (tid < 2) a.tally.all[tid] = 0;
    }
}

template <typename T, int G, int Q, bool SIGMOID, bool WHOLE>
static int launch_balance(BalanceArgs a, cudaStream_t st)
{
    const int64_t many = a.nseq * a.ncols, words = many + 2 * a.nseq;
    if (words <= SMALL_COUNTS && a.nrows * a.ncols <= SMALL_ELEMENTS && a.nrows * 4 < SMALL_ELEMENTS) {
        int ranks = 1;
        while (ranks < MOST_CLUSTER && a.nrows * a.ncols > (int64_t)ranks * 4096) ranks *= 2;
        return launch_cluster(balance_small_kernel<T, G, Q, SIGMOID, WHOLE>, (unsigned)ranks, ranks, BT, 0, 0, st, a);
    }
    constexpr int AT_ONCE = BW * 32 / G;
    const int64_t most = (int64_t)sm_count() * 8;
    const int64_t grid = max((int64_t)1, min((int64_t)sm_count() * balance_ctas<T, Q>(), ceil_div(a.nrows, AT_ONCE * 2)));
    void *room = nullptr;
    a.kept = words <= KEPT_COUNTS;
    CB_TRY(scratch(SLOT_MISC, (size_t)most * sizeof(double) + (a.kept ? 0 : (size_t)(2 + 2 * a.nseq) * sizeof(u64)), &room));
    a.partial = (double *)room;
    if (a.kept) {
        u64 *kept = nullptr;
        CB_CUDA(cudaGetSymbolAddress((void **)&kept, g_kept));
        a.tally = {kept, kept + many, kept + many + 2 * a.nseq};
    } else {
        u64 *info = (u64 *)(a.partial + most);
        a.tally = {(u64 *)a.counts, info, info + 2 * a.nseq};
        CB_CUDA(cudaMemsetAsync(a.counts, 0, (size_t)many * sizeof(int64_t), st));
        CB_CUDA(cudaMemsetAsync(info, 0, (size_t)(2 + 2 * a.nseq) * sizeof(u64), st));
    }
    const int64_t per = max((int64_t)BT, ceil_div(ceil_div(a.nrows, most), BT) * BT);
    if (a.nrows > 0) balance_count_kernel<<<(unsigned)ceil_div(a.nrows, per), BT, 0, st>>>(a, per);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) e = launch_behind(balance_kernel<T, G, Q, SIGMOID, WHOLE>, dim3((unsigned)grid), BT, 0, st, a);
    if (e != cudaSuccess) {
        if (a.kept) cudaMemsetAsync(a.tally.counts, 0, sizeof(g_kept), st);       // what was counted is not the next call's
        return fail("balance_loss: launch failed: %s", cudaGetErrorString(e));
    }
    return 0;
}

template <typename T, int G, int Q, bool SIGMOID>
static int launch_balance(const BalanceArgs &a, cudaStream_t st)
{
    return a.whole ? launch_balance<T, G, Q, SIGMOID, true>(a, st) : launch_balance<T, G, Q, SIGMOID, false>(a, st);
}

// G lanes x Q granules of N elements just cover the experts
template <typename T, bool SIGMOID>
static int dispatch_balance(const BalanceArgs &a, cudaStream_t st)
{
    const int granules = (a.ncols + Granule<T>::N - 1) / Granule<T>::N;
    if (granules <= 1) return launch_balance<T, 1, 1, SIGMOID>(a, st);
    if (granules <= 2) return launch_balance<T, 2, 1, SIGMOID>(a, st);
    if (granules <= 4) return launch_balance<T, 4, 1, SIGMOID>(a, st);
    if (granules <= 8) return launch_balance<T, 8, 1, SIGMOID>(a, st);
    if (granules <= 16) return launch_balance<T, 16, 1, SIGMOID>(a, st);
    if (granules <= 32) return launch_balance<T, 32, 1, SIGMOID>(a, st);
    if (granules <= 64) return launch_balance<T, 32, 2, SIGMOID>(a, st);
    if (granules <= 128) return launch_balance<T, 32, 4, SIGMOID>(a, st);
    return launch_balance<T, 32, 1024 / (32 * Granule<T>::N), SIGMOID>(a, st);
}

template <typename T>
static int balance_loss(int64_t nrows, int64_t ncols, const int64_t *pos, const int64_t *crd, int64_t nseq, const int64_t *seq, const uint8_t *mask,
                        int32_t sigmoid, const void *r, int64_t ldr, void *grad, int64_t ldg, const double *scale, int64_t *counts, float *loss,
                        void *stream)
{
    clear_error();
    cudaStream_t st = (cudaStream_t)stream;
    if (nrows < 0 || ncols <= 0) return fail("balance_loss: %lld rows of %lld columns", (long long)nrows, (long long)ncols);
    if (ncols > MOST_EXPERTS) return fail("balance_loss: %lld experts; at most %d", (long long)ncols, MOST_EXPERTS);
    if (ldr < ncols || (grad && ldg < ncols)) return fail("balance_loss: leading dimension smaller than the number of columns");
    if (nseq < 1 || (nseq > 1 && !seq)) return fail("balance_loss: %lld sequences without their bounds", (long long)nseq);
    if ((uintptr_t)r % sizeof(T) || (uintptr_t)grad % sizeof(T)) return fail("balance_loss: an address that is not a multiple of the element's size");
    const int64_t size = (int64_t)sizeof(T);
    const bool whole = ncols * size % 16 == 0 && ((uintptr_t)r | (uintptr_t)grad) % 16 == 0 && ldr * size % 16 == 0 && ldg * size % 16 == 0;
    const BalanceArgs a = {nrows, (int)ncols, pos, crd, nseq, seq, mask, r, ldr, grad, ldg, (float)*scale, whole, {}, false, counts, nullptr, loss,
                           next_counter()};
    if (!a.counter) return 1;
    return sigmoid ? dispatch_balance<T, true>(a, st) : dispatch_balance<T, false>(a, st);
}

}  // namespace cb200

#define BALANCE(suffix, T)                                                                                                              \
    extern "C" int32_t comet_b200_dev_balance_loss_##suffix##_i64(                                                                       \
        int64_t nrows, int64_t ncols, const int64_t *pos, const int64_t *crd, int64_t nseq, const int64_t *seq, const uint8_t *mask,     \
        int32_t sigmoid, const void *r, int64_t ldr, void *grad, int64_t ldg, const double *scale, int64_t *counts, float *loss,         \
        void *stream)                                                                                                                    \
    {                                                                                                                                    \
        return cb200::balance_loss<T>(nrows, ncols, pos, crd, nseq, seq, mask, sigmoid, r, ldr, grad, ldg, scale, counts, loss, stream); \
    }
BALANCE(bf16, __nv_bfloat16)
BALANCE(f16, __half)
BALANCE(f32, float)
