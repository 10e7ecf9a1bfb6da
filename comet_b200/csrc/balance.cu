// The balance loss of a router: S (CSR, rows tokens, columns experts) says which experts took which tokens, R are the router's
// logits.  A row is active if it stores something and its mask is not 0.  With N active rows and K entries in a sequence,
// f_e = (entries in column e) / K and P_e = the mean over active rows of p_e, p = softmax(R) or sigmoid(R) / sum sigmoid(R):
//   loss = scale * (mean over sequences with active rows of  E * sum_e f_e P_e)
//   d loss / d r_e = scale E / (sequences N) * p_e (f_e - sum_j f_j p_j)          [times (1 - sigmoid(r_e))]
// The counts are all that the gradient needs of other rows, so they come first and R is read once.  f is used as
// g = f - 1 / E, taken from whole numbers: for balanced experts the difference f_e - sum f p would lose its digits otherwise.
// sigmoid(r) / sum is softmax(log sigmoid(r)), which holds where every sigmoid underflows.
//
// Bound: HBM, R and its gradient; small batches: the launches.
#include "logits.cuh"
#include "stream.cuh"

namespace cb200 {

static const int BT = 256, MOST_EXPERTS = 1024;

// What the counts leave for the main kernel, in SLOT_MISC: {sequences with active rows, -}, then {active rows, entries} per sequence.
typedef unsigned long long u64;

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

__global__ void __launch_bounds__(BT)
balance_count_kernel(int64_t nrows, int ncols, const int64_t *__restrict__ pos, const int64_t *__restrict__ crd, int64_t nseq,
                     const int64_t *__restrict__ seq, const uint8_t *__restrict__ mask, u64 *__restrict__ counts, u64 *__restrict__ info)
{
    for (int64_t t = (int64_t)blockIdx.x * BT + threadIdx.x; t < nrows; t += (int64_t)gridDim.x * BT) {
        const int64_t lo = pos[t], hi = pos[t + 1];
        if (lo >= hi || (mask && !mask[t])) continue;
        const int64_t s = seq ? sequence_of(seq, nseq, t) : 0;
        for (int64_t e = lo; e < hi; e++) {
            const int64_t j = crd[e];
            if (j >= 0 && j < ncols) atomicAdd(&counts[s * ncols + j], 1ull);
            else atomicExch(&info[1], 1ull);
        }
        if (atomicAdd(&info[2 + 2 * s], 1ull) == 0) atomicAdd(&info[0], 1ull);
        atomicAdd(&info[3 + 2 * s], (u64)(hi - lo));
    }
}

struct BalanceArgs {
    int64_t nrows;
    int ncols;
    const int64_t *pos;
    int64_t nseq;
    const int64_t *seq;
    const uint8_t *mask;
    const void *r;
    int64_t ldr;
    void *grad;
    int64_t ldg;
    float scale;
    const u64 *counts, *info;
    double *partial;
    float *loss;
    unsigned *counter;
};

// A warp per row, a lane's experts 32 apart.
template <typename T, int R, bool SIGMOID>
__global__ void __launch_bounds__(BT)
balance_kernel(const BalanceArgs a)
{
    const int lane = threadIdx.x & 31;
    const float sequences = (float)a.info[0];
    double sum = 0.0;
    for (int64_t t = ((int64_t)blockIdx.x * BT + threadIdx.x) >> 5; t < a.nrows; t += ((int64_t)gridDim.x * BT) >> 5) {
        const T *r = (const T *)a.r + t * a.ldr;
        T *grad = a.grad ? (T *)a.grad + t * a.ldg : nullptr;
        if (a.pos[t] >= a.pos[t + 1] || (a.mask && !a.mask[t])) {
            if (grad)
                for (int e = lane; e < a.ncols; e += 32) grad[e] = from_float<T>(0.0f);
            continue;
        }
        const int64_t s = a.seq ? sequence_of(a.seq, a.nseq, t) : 0;
        const float rows = (float)a.info[2 + 2 * s], by = a.scale * (float)a.ncols / (sequences * rows);
        const u64 entries = a.info[3 + 2 * s];
        const float unit = (float)(1.0 / ((double)entries * a.ncols));
        float u[R], slope[R], m = MINUS_INF;
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int e = lane + 32 * i;
            u[i] = e < a.ncols ? to_float(r[e]) : MINUS_INF;
            slope[i] = 1.0f;
            if (SIGMOID) {
                const float d = expf(-fabsf(u[i])), l = fminf(u[i], 0.0f) - log1pf(d);
                slope[i] = u[i] > 0.0f ? d / (1.0f + d) : 1.0f / (1.0f + d);       // 1 - sigmoid
                u[i] = u[i] == MINUS_INF ? MINUS_INF : l;
            }
            m = max_nan(m, u[i]);
        }
        m = warp_max(m);
        float p = 0.0f, gp = 0.0f, g[R];
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int e = lane + 32 * i;
            g[i] = e < a.ncols ? (float)((int64_t)a.counts[s * a.ncols + e] * a.ncols - (int64_t)entries) * unit : 0.0f;
            u[i] = m == MINUS_INF ? 0.0f : exp2_fast((u[i] - m) * LOG2E);
            p += u[i];
            gp += u[i] * g[i];
        }
        p = warp_sum(p);
        gp = warp_sum(gp);
        const float inv = p == 0.0f ? 0.0f : 1.0f / p;
        gp *= inv;
        if (grad)
#pragma unroll
            for (int i = 0; i < R; i++) {
                const int e = lane + 32 * i;
                if (e < a.ncols) grad[e] = from_float<T>(by * (u[i] * inv) * (g[i] - gp) * slope[i]);
            }
        if (p != 0.0f) sum += (double)by * (1.0f / (float)a.ncols + gp);
    }
    __shared__ double sums[BT / 32];
    __shared__ bool last;
    if (lane == 0) sums[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < BT / 32; i++) sum += sums[i];
        a.partial[blockIdx.x] = sum;
        last = last_of(a.counter, gridDim.x);
    }
    __syncthreads();
    if (!last || threadIdx.x >= 32) return;
    __threadfence();
    sum = 0.0;
    for (int i = lane; i < (int)gridDim.x; i += 32) sum += __ldcg(a.partial + i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) *a.loss = a.info[1] ? __int_as_float(0x7fffffff) : (float)sum;
}

template <typename T, bool SIGMOID>
static void launch_balance(const BalanceArgs &a, unsigned grid, cudaStream_t st)
{
    if (a.ncols <= 32) balance_kernel<T, 1, SIGMOID><<<grid, BT, 0, st>>>(a);
    else if (a.ncols <= 64) balance_kernel<T, 2, SIGMOID><<<grid, BT, 0, st>>>(a);
    else if (a.ncols <= 128) balance_kernel<T, 4, SIGMOID><<<grid, BT, 0, st>>>(a);
    else if (a.ncols <= 256) balance_kernel<T, 8, SIGMOID><<<grid, BT, 0, st>>>(a);
    else if (a.ncols <= 512) balance_kernel<T, 16, SIGMOID><<<grid, BT, 0, st>>>(a);
    else balance_kernel<T, 32, SIGMOID><<<grid, BT, 0, st>>>(a);
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
    const int64_t most = (int64_t)sm_count() * 8;
    int64_t grid = ceil_div(nrows, BT / 32);
    if (grid > most) grid = most;
    if (grid < 1) grid = 1;
    void *room = nullptr;
    CB_TRY(scratch(SLOT_MISC, (size_t)(2 + 2 * nseq) * sizeof(u64) + (size_t)most * sizeof(double), &room));
    u64 *info = (u64 *)room;
    BalanceArgs a = {nrows, (int)ncols, pos, nseq, seq, mask, r, ldr, grad, ldg, (float)*scale, (const u64 *)counts, info, (double *)(info + 2 + 2 * nseq),
                     loss, next_counter()};
    if (!a.counter) return 1;
    CB_CUDA(cudaMemsetAsync(counts, 0, (size_t)(nseq * ncols) * sizeof(int64_t), st));
    CB_CUDA(cudaMemsetAsync(info, 0, (size_t)(2 + 2 * nseq) * sizeof(u64), st));
    int64_t blocks = ceil_div(nrows, BT);
    if (blocks > most) blocks = most;
    if (blocks > 0) balance_count_kernel<<<(unsigned)blocks, BT, 0, st>>>(nrows, (int)ncols, pos, crd, nseq, seq, mask, (u64 *)counts, info);
    CB_LAUNCH_CHECK();
    if (sigmoid) launch_balance<T, true>(a, (unsigned)grid, st);
    else launch_balance<T, false>(a, (unsigned)grid, st);
    CB_LAUNCH_CHECK();
    return 0;
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
