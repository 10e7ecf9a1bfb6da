// Shared by the operators on rows of logits (top.cu, distill.cu, balance.cu): the three element types, 16-byte vectors of
// them, and sums and maxima over a CTA.  Arithmetic is in f32 whatever the type; a result is rounded once, when it is stored.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace cb200 {

static const int MOST_CLUSTER = 8;                  // CTAs of a cluster that every device takes
static const double LOG2E_D = 1.4426950408889634;
// 1 / temperature and log2(e) / temperature are f32 numbers
inline bool temperature_fits(double t) { return t >= 1e-38 && t <= 1e30; }

#ifdef __CUDACC__
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float MINUS_INF = -__builtin_huge_valf();
// (x - m) c as x c - (m c) is off by the rounding of m c, the same for all x: a factor of less than 2^(1/4) up to here, and beyond f32 from 2^31 on.
constexpr float NEAR = 4194304.0f;

__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_float(float v) { return v; }

__device__ __forceinline__ float min_nan(float a, float b)
{
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// 1 / v, correct to one unit in the last place; 0 from 2^126 on
__device__ __forceinline__ float reciprocal(float v)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
typedef unsigned long long u64_pair;

// a NaN among the operands is the result
__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ double max_nan(double a, double b) { return a != a || a > b ? a : b; }

// two f32 operations in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(*(u64_pair *)&r) : "l"(*(const u64_pair *)&a), "l"(*(const u64_pair *)&b));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(*(u64_pair *)&r) : "l"(*(const u64_pair *)&a), "l"(*(const u64_pair *)&b));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(*(u64_pair *)&r)
        : "l"(*(const u64_pair *)&a), "l"(*(const u64_pair *)&b), "l"(*(const u64_pair *)&c));
    return r;
}

// 16 bytes of elements
template <typename T>
struct Granule;
template <>
struct Granule<float> {
    static constexpr int N = 4;
    uint4 w;
    static __device__ __forceinline__ Granule least() { return {make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u)}; }          // -inf
    __device__ __forceinline__ void unpack(float2 (&v)[2]) const
    {
        v[0] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
        v[1] = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
    }
    typedef float Most;                            // a granule's largest element, for 16-bit types of the even and of the odd ones
    __device__ __forceinline__ Most most() const
    {
        return max_nan(max_nan(__uint_as_float(w.x), __uint_as_float(w.y)), max_nan(__uint_as_float(w.z), __uint_as_float(w.w)));
    }
    // a bit per element that is not smaller than `than` (a NaN never is, nor is anything smaller than one)
    __device__ __forceinline__ unsigned at_least(float than) const
    {
        return (__uint_as_float(w.x) < than ? 0u : 1u) | (__uint_as_float(w.y) < than ? 0u : 2u) | (__uint_as_float(w.z) < than ? 0u : 4u) |
               (__uint_as_float(w.w) < than ? 0u : 8u);
    }
    __device__ __forceinline__ void unpack(float (&v)[4]) const
    {
        v[0] = __uint_as_float(w.x);
        v[1] = __uint_as_float(w.y);
        v[2] = __uint_as_float(w.z);
        v[3] = __uint_as_float(w.w);
    }
    __device__ __forceinline__ void pack(const float2 (&v)[2])
    {
        w = make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
    }
    __device__ __forceinline__ void pack(const float (&v)[4])
    {
        w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};
// a bit per element that is not smaller than `than`
template <typename T2>
__device__ __forceinline__ unsigned at_least16(const uint4 &w, T2 than)
{
    const unsigned v = (__hgeu2_mask(*(const T2 *)&w.x, than) & 0x00020001u) | (__hgeu2_mask(*(const T2 *)&w.y, than) & 0x00080004u) |
                       (__hgeu2_mask(*(const T2 *)&w.z, than) & 0x00200010u) | (__hgeu2_mask(*(const T2 *)&w.w, than) & 0x00800040u);
    return (v | v >> 16) & 0xffu;
}
template <>
struct Granule<__nv_bfloat16> {
    static constexpr int N = 8;
    uint4 w;
    static __device__ __forceinline__ Granule least() { return {make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u)}; }          // -inf
    __device__ __forceinline__ void unpack(float2 (&v)[4]) const
    {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
    }
    typedef __nv_bfloat162 Most;
    __device__ __forceinline__ Most most() const
    {
        return __hmax2_nan(__hmax2_nan(*(const Most *)&w.x, *(const Most *)&w.y), __hmax2_nan(*(const Most *)&w.z, *(const Most *)&w.w));
    }
    __device__ __forceinline__ unsigned at_least(__nv_bfloat16 than) const { return at_least16<__nv_bfloat162>(w, {than, than}); }
    __device__ __forceinline__ void unpack(float (&v)[8]) const
    {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = __uint_as_float(u[i] << 16);
            v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
    __device__ __forceinline__ void pack(const float2 (&v)[4])
    {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 p = __floats2bfloat162_rn(v[i].x, v[i].y);
            u[i] = *(const uint32_t *)&p;
        }
        w = make_uint4(u[0], u[1], u[2], u[3]);
    }
    __device__ __forceinline__ void pack(const float (&v)[8])
    {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            u[i] = *(const uint32_t *)&p;
        }
        w = make_uint4(u[0], u[1], u[2], u[3]);
    }
};
template <>
struct Granule<__half> {
    static constexpr int N = 8;
    uint4 w;
    static __device__ __forceinline__ Granule least() { return {make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u)}; }          // -inf
    __device__ __forceinline__ void unpack(float2 (&v)[4]) const
    {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __half22float2(*(const __half2 *)&u[i]);
    }
    typedef __half2 Most;
    __device__ __forceinline__ Most most() const
    {
        return __hmax2_nan(__hmax2_nan(*(const Most *)&w.x, *(const Most *)&w.y), __hmax2_nan(*(const Most *)&w.z, *(const Most *)&w.w));
    }
    __device__ __forceinline__ unsigned at_least(__half than) const { return at_least16<__half2>(w, {than, than}); }
    __device__ __forceinline__ void unpack(float (&v)[8]) const
    {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*(const __half2 *)&u[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
    __device__ __forceinline__ void pack(const float2 (&v)[4])
    {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __half2 p = __floats2half2_rn(v[i].x, v[i].y);
            u[i] = *(const uint32_t *)&p;
        }
        w = make_uint4(u[0], u[1], u[2], u[3]);
    }
    __device__ __forceinline__ void pack(const float (&v)[8])
    {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __half2 p = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            u[i] = *(const uint32_t *)&p;
        }
        w = make_uint4(u[0], u[1], u[2], u[3]);
    }
};

// largest elements: NaN if one is
__device__ __forceinline__ float most_of(float a, float b) { return max_nan(a, b); }
__device__ __forceinline__ __nv_bfloat162 most_of(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmax2_nan(a, b); }
__device__ __forceinline__ __half2 most_of(__half2 a, __half2 b) { return __hmax2_nan(a, b); }
__device__ __forceinline__ float largest(float a) { return a; }
__device__ __forceinline__ __nv_bfloat16 largest(__nv_bfloat162 a) { return __hmax_nan(a.x, a.y); }
__device__ __forceinline__ __half largest(__half2 a) { return __hmax_nan(a.x, a.y); }
// one of the elements is not smaller
__device__ __forceinline__ bool reaches(float a, float than) { return !(a < than); }
__device__ __forceinline__ bool reaches(__nv_bfloat162 a, __nv_bfloat16 than) { return __hgeu2_mask(a, {than, than}) != 0; }
__device__ __forceinline__ bool reaches(__half2 a, __half than) { return __hgeu2_mask(a, {than, than}) != 0; }

// 2^v, correct to two units in the last place; results below 2^-126 are 0
__device__ __forceinline__ float exp2_fast(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v)
{
    float r;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ double warp_max(double v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// N values per thread to their sums (or maxima) over the CTA, in every thread.  `room` holds N * WARPS floats and is free
// again after the next barrier.  Every thread adds in the same order: all have the same bits.
template <int N, int WARPS, bool MAX>
__device__ __forceinline__ void cta_reduce(float (&v)[N], float *room)
{
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = MAX ? warp_max(v[i]) : warp_sum(v[i]);
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; i++) room[i * WARPS + (threadIdx.x >> 5)] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        float s = room[i * WARPS];
#pragma unroll
        for (int w = 1; w < WARPS; w++) s = MAX ? max_nan(s, room[i * WARPS + w]) : s + room[i * WARPS + w];
        v[i] = s;
    }
}

__device__ __forceinline__ void copy_granule(void *to, const void *from)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
// 16 bytes, from and to BYTES behind the addresses
template <int BYTES>
__device__ __forceinline__ void copy_far(uint32_t to, const void *from)
{
    asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %2], 16;" ::"r"(to), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ unsigned cluster_size()
{
    unsigned r;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned cluster_rank()
{
    unsigned r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
template <typename V>
__device__ __forceinline__ uint32_t peer_address(const V *mine, unsigned rank)
{
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
    return at;
}
__device__ __forceinline__ void store_peer(float *mine, unsigned rank, float v)
{
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(peer_address(mine, rank)), "f"(v) : "memory");
}
__device__ __forceinline__ void store_peer(double *mine, unsigned rank, double v)
{
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(peer_address(mine, rank)), "d"(v) : "memory");
}
__device__ __forceinline__ float peer_load(const float *mine, unsigned rank)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer_address(mine, rank)) : "memory");
    return v;
}
__device__ __forceinline__ int peer_load(const int *mine, unsigned rank)
{
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(peer_address(mine, rank)) : "memory");
    return v;
}
__device__ __forceinline__ unsigned long long peer_load(const unsigned long long *mine, unsigned rank)
{
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(peer_address(mine, rank)) : "memory");
    return v;
}

// One of the counters by which the last CTA of a launch finds out that it is the last.  Each goes back to 0 by itself
// (atomicInc); a call takes the next one of 1024.
__device__ __forceinline__ bool last_of(unsigned *counter, unsigned ctas)
{
    __threadfence();
    return atomicInc(counter, ctas - 1) == ctas - 1;
}

// `ctas` CTAs in clusters of `ranks`.  `most`: the dynamic shared memory of the kernel's largest call.  It is the limit in every call, so that a
// second host thread, on its way to another call, does not lower the limit between this one's setting and its launch.
template <typename... P, typename... A>
inline int launch_cluster(void (*kernel)(P...), unsigned ctas, int ranks, int threads, size_t smem, size_t most, cudaStream_t st, A... args)
{
    if (smem > 16 * 1024) CB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ranks;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    CB_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
    return 0;
}
#endif

unsigned *next_counter();      // device address (top.cu); null, with the error kept, if there is no device

}  // namespace cb200
