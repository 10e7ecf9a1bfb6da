// The fifth-generation tensor cores: tensor copies into shared memory, the matrix instruction with its accumulators in tensor memory,
// and bounded waits for both.
#pragma once
#include <cuda.h>

#include "common.cuh"

namespace cb200 {

// A tensor map of 16-bit elements, depth x rows x cols, contiguous, with boxes of box_rows rows of 64 columns, which are 128-byte rows in shared memory,
// swizzled (experts.cu).
int make_box_map(const char *what, const void *base, bool bf16, int64_t depth, int64_t rows, int64_t cols, int box_rows, CUtensorMap *map);

#ifdef __CUDACC__
__device__ __forceinline__ uint32_t smem_at(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(uint32_t bar, unsigned count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, unsigned bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool bar_try(uint32_t bar, unsigned parity)
{
    unsigned ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Waits for a phase; false after two seconds, or once another wait of the CTA has run out (*broken).  steps: of products that the phase takes beside that, 64 terms
// each; one takes 0.35 to 0.5 us, and has 4.  (Whoever waits for single steps finds within two seconds that they have stopped.)
__device__ __forceinline__ bool bar_wait(uint32_t bar, unsigned parity, volatile int *broken, int steps = 0)
{
    unsigned long long began = 0;
    for (;;) {
        // unrolled by the compiler: a loop of one look at a time let the products of gated_batch wait 2 % longer
        for (int i = 0; i < 64; i++)
            if (bar_try(bar, parity)) return true;
        if (*broken) return false;
        unsigned long long now;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
        if (!began) began = now;
        if (now - began > 2000000000ull + 4000ull * (unsigned)steps) {
            *broken = 1;
            return false;
        }
    }
}
// one thread of a warp that is together
__device__ __forceinline__ bool elect()
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r) : : "memory");
    return r != 0;
}

__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *map, int c, int r, int z, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(c), "r"(r), "r"(z), "r"(bar) : "memory");
}
// contiguous bytes, a multiple of 16
__device__ __forceinline__ void load_bytes(uint32_t dst, const void *src, unsigned bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// 16 bytes, or zeros where `on` is not
__device__ __forceinline__ void copy_or_zero(uint32_t dst, const void *src, bool on)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
// the thread arrives at the barrier when its copies so far have landed
__device__ __forceinline__ void copies_to(uint32_t bar)
{
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
// what threads have written to shared memory, and this thread knows of, is seen by products issued from here on
__device__ __forceinline__ void shared_to_products() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// by a warp
__device__ __forceinline__ void tmem_alloc(uint32_t at, unsigned columns)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(at), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem, unsigned columns)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// An operand's tile in shared memory, 128-byte rows, 128-byte swizzle.  `lead`: bytes from one block of 64 rows of the product to the next where
// the rows of the tile are the sum's index (not looked at otherwise); `stride`: bytes from 8 rows of the tile to the next.
__device__ __forceinline__ uint64_t tile_descriptor(uint32_t at, unsigned lead, unsigned stride)
{
    return (uint64_t)((at & 0x3ffff) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// f32 sums of products of bf16 (or f16) numbers, m x n; rows_a, rows_b: the rows of the operand's tile are the sum's index
constexpr uint32_t product_descriptor(bool bf16, int m, int n, bool rows_a, bool rows_b)
{
    return 1u << 4 | (bf16 ? 1u : 0u) << 7 | (bf16 ? 1u : 0u) << 10 | (rows_a ? 1u : 0u) << 15 | (rows_b ? 1u : 0u) << 16 | (uint32_t)(n / 8) << 17 |
           (uint32_t)(m / 16) << 24;
}
__device__ __forceinline__ void product(uint32_t tmem, uint64_t a, uint64_t b, uint32_t kind, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem), "l"(a), "l"(b), "r"(kind), "r"((uint32_t)add) : "memory");
}
// the barrier's phase ends when the products issued so far are done
__device__ __forceinline__ void products_to(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// 16 or 32 columns of the warp's 32 rows, a row a thread.  The wait is part of it: only so does the compiler know that nothing may use the values before.
__device__ __forceinline__ void tmem_load(uint32_t at, float (&v)[16])
{
    uint32_t r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at) : "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_load(uint32_t at, float (&v)[32])
{
    uint32_t r[32];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(at) : "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}
#endif

}  // namespace cb200
