// Shared by the two kernels of the distillation loss (distill.cu: a cluster per row; distill_rows.cu: a CTA per row).
#pragma once
#include "logits.cuh"
#include "stream.cuh"

namespace cb200 {

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
    unsigned *counter;           // null: another kernel adds the rows up
};

// (x - m) c.  As x c - m c it is one operation, and the rounding of m c is a factor that all of a row's terms and their sum
// have alike; m c may be beyond f32 where the difference is not.
struct Exponent {
    float c, m, mc;
    bool near;
    __device__ __forceinline__ Exponent(float most, float c_) : c(c_), m(most == MINUS_INF ? 0.0f : most)
    {
        mc = m * c;
        near = fabsf(mc) < 1e30f;
    }
    __device__ __forceinline__ float of(float x) const { return near ? fmaf(x, c, -mc) : (x - m) * c; }
    __device__ __forceinline__ float2 of(float2 x) const { return fma2(x, make_float2(c, c), make_float2(-mc, -mc)); }      // near
    __device__ __forceinline__ float to(const Exponent &o) const { return near && o.near ? mc - o.mc : (m - o.m) * c; }
};

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

// The same loss by a CTA per row (distill_rows.cu); for batches that fill the chip.
template <typename T>
int distill_by_rows(DistillArgs a, int val_bytes, cudaStream_t st);

}  // namespace cb200
