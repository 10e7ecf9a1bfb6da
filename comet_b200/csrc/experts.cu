// The feed-forward block of a router's experts.  A CSR matrix says which rows of x (tokens) go to which experts; its entries e = (t, j) have a row each
// in h.  With w = [gate; up] of expert j (2 inner x width) and v (width x inner):
//   gated     h_e = act(gate x_t) * (up x_t)                 dz_e = [dh_e * up x_t * act'(gate x_t), dh_e * act(gate x_t)]
//                                                            dx_t = sum_e w' dz_e,  dw_j = sum_e dz_e x_t'
//   combine   y_t = sum_e val_e v h_e                        dval_e = h_e (v' dy_t),  dh_e = val_e v' dy_t,  dv_j = sum_e val_e dy_t h_e'
// act(g) = g s(u) with the logistic function s, u = g for silu and 2 sqrt(2 / pi) (g + 0.044715 g^3) for gelu (its tanh form).
//
// All of these are one kernel: tiles of 128 x 256 sums in tensor memory, 64 terms a step, with the operands' tiles in a ring in shared memory.  One warp
// fetches by tensor copies, four by row numbers, one issues the products, eight take the sums of the tile before out of tensor memory.  Weights, and what a
// kernel before has left in the order of the slots (dz, val h), come by tensor copies; rows of x, h and dy by their number, 16 bytes a copy, so that
// nothing is sorted first.  (A tensor copy of four numbered rows takes about 70 clocks whatever their width: 65536 entries of width 2048 by 64 experts of
// inner 1024, the gated product, 1200 us with them, 438 without.)
//
// Bound: for that product, 550 GFLOP, 440 to 470 us when the chip is cool and 530 in a row of passes, where the power cap leaves 1.5 GHz (a library's plain product of the
// same size: 370 and 430).  Tensor cores are active 70 to 72 % of the clocks: a step of 64 terms is 512 clocks of theirs and takes some 708, start and end of the launch
// included.  The operands' 48 KB a step come into an SM at 65.5 bytes a clock over the whole launch (dx 60, dz 56), so the way from the L2 to an SM is the
// likely bound; shared memory's banks are read in 28 % of the clocks and written in 27 %, the L2 is busy 36 %.  Where sums are short (dw: 7 steps a
// tile, active 44 %; dv 45 %) or their results f32 (combine, 52 %), the results' bytes.
// Three forms:
//   ROWS   rows of a tile's tokens, times a weight whose rows are outputs                (forward passes, dz)
//   BACK   the same, times a weight whose rows are the sum's index                       (dx, v' dy)
//   OUTER  sums over an expert's tokens of two rows                                      (dw, dv)
// Sums of a token's experts go through f32 rows, one for each entry, and are added in the entries' order: the same bits in every call.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <string.h>

#include <atomic>
#include <type_traits>

#include "groups.cuh"
#include "logits.cuh"
#include "stream.cuh"
#include "tensor.cuh"

namespace cb200 {

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static int make_map(const char *what, const void *base, bool bf16, int rank, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box,
                    CUtensorMap *map)
{
    static std::atomic<EncodeTiled> found{nullptr};            // the driver's, the same for every device; two threads may look for it at once
    EncodeTiled encode = found.load();
    if (!encode) {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess || !fn || q != cudaDriverEntryPointSuccess)
            return fail("%s: cuTensorMapEncodeTiled is not available from this driver", what);
        encode = (EncodeTiled)fn;
        found.store(encode);
    }
    const cuuint32_t ones[3] = {1, 1, 1};
    const CUresult r = encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, (void *)base, dims, strides, box, ones,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : fail("%s: cuTensorMapEncodeTiled refused a map (error %d)", what, (int)r);
}

int make_box_map(const char *what, const void *base, bool bf16, int64_t depth, int64_t rows, int64_t cols, int box_rows, CUtensorMap *map)
{
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)depth}, strides[2] = {(cuuint64_t)cols * 2, (cuuint64_t)(cols * rows) * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
    return make_map(what, base, bf16, 3, dims, strides, box, map);
}

enum Form { ROWS, BACK, OUTER };
enum Sums { GATED, GATED_GRAD, ENTRY_ROWS, COMBINE_GRAD, WEIGHT };

// A tile has 128 rows and W columns: 256, or, where those are few for the chip, 64, two CTAs on an SM (launch_shape).
static const int TM = 128, WIDE = 256, NARROW = 64, TK = 64;
static const int A_BYTES = TM * TK * 2;
static const int TAKERS = 256, FETCHERS = 128, PRODUCT_THREADS = TAKERS + FETCHERS + 64;
template <int W>
struct Shape {
    static constexpr int B_BYTES = W * TK * 2, STEP = A_BYTES + B_BYTES, RING = 4;
    static constexpr int TAKEN = W == WIDE ? 128 : 32;         // bytes of a row that a warp takes out at a time
    static constexpr int SMEM = RING * STEP + TAKERS * TAKEN + 1024;
};
// The tensor cores cut off what does not fit into an f32 sum, each time that they add, so long sums are off by more than f32 sums are.  In results of 16 bits that is
// nothing; d_values is f32, and was off by 2.0e-6 of its norm at a width of 2048, 9.1e-6 at 8192.  There a tile's sums are taken out after so many steps and added up,
// rounded to the nearest, in the takers' registers (0: not at all): 4.8e-7 at any width after 8 steps, 1.0e-6 after 16, 2.6e-7 after 4; f32 products 2e-7 to 4e-7.
// While the takers are at a tile's results, products for two such segments can go on: v'dy of combine_grad_step 97 us after 8 steps, 89 after 16, 106 after 4, 86 not at all.
constexpr int segment(int sums) { return sums == COMBINE_GRAD ? 8 : 0; }
// In a wide tile that is 128 sums a thread.  The takers get the registers that the other warps do not use: of the 128 that each of 512 threads starts with, theirs then
// have 192 and the others' 64, by warpgroups of 128 threads.
constexpr bool many_registers(int w, int sums) { return w == WIDE && segment(sums); }
constexpr int product_threads(int w, int sums) { return many_registers(w, sums) ? 512 : PRODUCT_THREADS; }
static_assert(TAKERS * 192 + (512 - TAKERS) * 64 <= 512 * 128 && TAKERS % 128 == 0, "registers that are given were there");

struct ProductArgs {
    Groups g;
    const int *numbers;              // of each slot's row of the operand that is fetched by rows
    const void *numbered;            // that operand: its rows, their stride, and their columns
    int64_t ld;
    int numbered_cols;
    int terms;                       // of the sums (not OUTER)
    int tiles_m, tiles_n;            // tiles of a weight's rows (OUTER), tiles of columns
    int rows, cols;                  // of an expert's result (OUTER), of a result row
    int64_t nnz;
    bool gelu;
    const void *other;               // dh, h
    const float *val;
    void *out, *scaled;              // 16-bit results; val * h
    float *sums;                     // rows of f32, or sums of products per tile of columns

    void number(const int *list, const void *rows, int64_t stride, int64_t n)
    {
        numbers = list;
        numbered = rows;
        ld = stride;
        numbered_cols = (int)n;
    }
};

struct Tile {
    int m, n, group, steps, slot;    // slot: the first one
    int half;                        // 0: all of the tile's columns, 1 or 2: the first or the second half of them
};

__device__ __forceinline__ float logistic(float u) { return __fdividef(1.0f, 1.0f + exp2_fast(-LOG2E * u)); }
// what s() takes, and its slope
__device__ __forceinline__ float2 gate_of(float g, bool gelu)
{
    constexpr float A = 1.5957691216057308f, B = 0.044715f;                          // 2 sqrt(2 / pi)
    return gelu ? make_float2(A * fmaf(B * g * g, g, g), A * fmaf(3.0f * B * g, g, 1.0f)) : make_float2(g, 1.0f);
}

template <typename T>
__device__ __forceinline__ void store8(T *to, const float *v)
{
    Granule<T> out;
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = v[i];
    out.pack(f);
    *(uint4 *)to = out.w;
}
template <typename T>
__device__ __forceinline__ void load8(float *v, const T *from)
{
    Granule<T> in;
    in.w = *(const uint4 *)from;
    float f[8];
    in.unpack(f);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = f[i];
}

// A warp's 32 rows of BYTES bytes in shared memory, on their way to or from global memory: a thread has a row, but reads and writes of global memory are
// of whole rows, BYTES / 16 neighbouring lanes each.  (Stores by the threads of the rows touch 32 lines an instruction: the sums of combine_batch
// were taken out in twice the time of the products.)
template <typename E, int BYTES>
struct Stage {
    static constexpr int LANES = BYTES / 16, N = 16 / sizeof(E), COLS = BYTES / sizeof(E);
    unsigned char *room;
    int lane;
    __device__ __forceinline__ uint4 &at(int row, int chunk) const { return *(uint4 *)(room + row * BYTES + ((chunk ^ (row & (LANES - 1))) << 4)); }
    __device__ __forceinline__ void put(int chunk, const float *v) const
    {
        Granule<E> out;
        float f[N];
#pragma unroll
        for (int i = 0; i < N; i++) f[i] = v[i];
        out.pack(f);
        at(lane, chunk) = out.w;
    }
    __device__ __forceinline__ void get(int chunk, float *v) const
    {
        Granule<E> in;
        in.w = at(lane, chunk);
        float f[N];
        in.unpack(f);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = f[i];
    }
    // rows from base + first (each thread's own; negative: none), `cols` of them there
    __device__ __forceinline__ void out(E *base, int64_t first, int cols) const
    {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < LANES; i++) {
            const int row = i * (32 / LANES) + lane / LANES, chunk = lane % LANES;
            const int64_t to = __shfl_sync(0xffffffffu, first, row);
            if (to >= 0 && chunk * N < cols) *(uint4 *)(base + to + chunk * N) = at(row, chunk);
        }
        __syncwarp();
    }
    __device__ __forceinline__ void in(const E *base, int64_t first, int cols) const
    {
#pragma unroll
        for (int i = 0; i < LANES; i++) {
            const int row = i * (32 / LANES) + lane / LANES, chunk = lane % LANES;
            const int64_t from = __shfl_sync(0xffffffffu, first, row);
            at(row, chunk) = from >= 0 && chunk * N < cols ? *(const uint4 *)(base + from + chunk * N) : make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
    }
    // in two steps: on their way, and there
    __device__ __forceinline__ void fetch(const E *base, int64_t first, int cols) const
    {
#pragma unroll
        for (int i = 0; i < LANES; i++) {
            const int row = i * (32 / LANES) + lane / LANES, chunk = lane % LANES;
            const int64_t from = __shfl_sync(0xffffffffu, first, row);
            const bool there = from >= 0 && chunk * N < cols;
            copy_or_zero(smem_at(&at(row, chunk)), base + (there ? from + chunk * N : 0), there);
        }
    }
    __device__ __forceinline__ void fetched() const
    {
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
    }
    // the same by way of registers
    __device__ __forceinline__ void load(uint4 (&v)[LANES], const E *base, int64_t first, int cols) const
    {
#pragma unroll
        for (int i = 0; i < LANES; i++) {
            const int64_t from = __shfl_sync(0xffffffffu, first, i * (32 / LANES) + lane / LANES);
            v[i] = from >= 0 && lane % LANES * N < cols ? *(const uint4 *)(base + from + lane % LANES * N) : make_uint4(0, 0, 0, 0);
        }
    }
    __device__ __forceinline__ void loaded(const uint4 (&v)[LANES]) const
    {
#pragma unroll
        for (int i = 0; i < LANES; i++) at(i * (32 / LANES) + lane / LANES, lane % LANES) = v[i];
        __syncwarp();
    }
};

// A tile's sums, by two warps for each 32 rows, a half of the columns each; tmem: tensor memory of the rows.  entry: that of the thread's row,
// negative if there is none.
template <typename T, int W, int SUMS>
__device__ __forceinline__ void take_sums(const ProductArgs &a, uint32_t tmem, bool none, const Tile &t, int half, int row, int64_t entry, unsigned char *room)
{
    constexpr int BYTES = Shape<W>::TAKEN;
    const Stage<T, BYTES> st = {room, (int)threadIdx.x & 31};
    if constexpr (SUMS == GATED || SUMS == GATED_GRAD) {
        constexpr int MINE = W / 4, PART = MINE < 32 ? MINE : 32;                    // columns of the warp, at a time
        static_assert(MINE == st.COLS, "one row of the stage");
        const int inner = a.cols, f0 = t.n * (W / 2) + half * MINE, left = inner - f0;
        if (left <= 0) return;
        const uint32_t at = tmem + half * MINE;
        if (SUMS == GATED) {
#pragma unroll
            for (int c = 0; c < MINE; c += PART) {
                float gate[PART], up[PART];
                tmem_load(at + c, gate);
                tmem_load(at + W / 2 + c, up);
#pragma unroll
                for (int i = 0; i < PART; i++) gate[i] = gate[i] * logistic(gate_of(gate[i], a.gelu).x) * up[i];
#pragma unroll
                for (int i = 0; i < PART; i += 8) st.put((c + i) / 8, gate + i);
            }
            st.out((T *)a.out, entry < 0 ? -1 : entry * inner + f0, left);
        } else {
            // PART columns at a time: with all 64 there are not registers enough
            const Stage<T, PART * 2> part = {room, (int)threadIdx.x & 31};
#pragma unroll 1
            for (int c = 0; c < MINE; c += PART) {
                float d[PART], gate[PART], up[PART];
                part.in((const T *)a.other, entry < 0 ? -1 : entry * inner + f0 + c, left - c);          // a row of zeros where there is none
#pragma unroll
                for (int i = 0; i < PART; i += 8) part.get(i / 8, d + i);
                tmem_load(at + c, gate);
                tmem_load(at + W / 2 + c, up);
#pragma unroll
                for (int i = 0; i < PART; i++) {
                    const float g = gate[i];
                    const float2 u = gate_of(g, a.gelu);
                    const float s = logistic(u.x);
                    const float curve = g * s * (1.0f - s);                          // 0 where gelu's u, and u's slope, may be infinite
                    gate[i] = d[i] * up[i] * (curve == 0.0f ? s : fmaf(curve, u.y, s));
                    up[i] = d[i] * g * s;
                }
                // Rounded to the operands' type, as the tensor cores take them: a step of that type in dx and dw beside the last one (2.3e-3 of a bf16 result's norm
                // instead of 1.7e-3).  In two parts of that type each they would be multiplied with W and X twice: dx and dw are more than half of the call.
                const int64_t to = (int64_t)(t.slot + row) * 2 * inner + f0 + c;
#pragma unroll
                for (int i = 0; i < PART; i += 8) part.put(i / 8, gate + i);
                part.out((T *)a.out, to, left - c);
#pragma unroll
                for (int i = 0; i < PART; i += 8) part.put(i / 8, up + i);
                part.out((T *)a.out, to + inner, left - c);
            }
        }
    } else if constexpr (SUMS == ENTRY_ROWS) {
        constexpr int MINE = W / 2, PART = BYTES / 4;
        const Stage<float, BYTES> rows = {room, (int)threadIdx.x & 31};
        const int c0 = t.n * W + half * MINE;
        const float by = entry >= 0 && a.val ? a.val[entry] : 1.0f;
#pragma unroll 1
        for (int c = 0; c < MINE; c += W == WIDE ? 32 : 16) {
            if (c0 + c >= a.cols) break;
            float v[W == WIDE ? 32 : 16];
            __syncwarp();
            tmem_load(tmem + half * MINE + c, v);
#pragma unroll
            for (int p = 0; p < (W == WIDE ? 32 : 16); p += PART) {
#pragma unroll
                for (int i = 0; i < PART; i++) v[p + i] *= by;
#pragma unroll
                for (int i = 0; i < PART; i += 4) rows.put(i / 4, v + p + i);
                rows.out(a.sums, entry < 0 ? -1 : entry * a.cols + c0 + c + p, a.cols - c0 - c - p);
            }
        }
    } else {
        constexpr int MINE = W / 2, PART = st.COLS < 32 ? st.COLS : 32;
        const int c0 = t.n * W + half * MINE, r = t.m * TM + row;
        const int64_t first = r < a.rows ? ((int64_t)t.group * a.rows + r) * a.cols + c0 : -1;
#pragma unroll 1
        for (int c = 0; c < MINE; c += st.COLS) {
            if (c0 + c >= a.cols) break;
            __syncwarp();
#pragma unroll
            for (int p = 0; p < st.COLS; p += PART) {
                float v[PART];
                if (none) {                        // an expert without tokens
#pragma unroll
                    for (int i = 0; i < PART; i++) v[i] = 0.0f;
                } else {
                    tmem_load(tmem + half * MINE + c + p, v);
                }
#pragma unroll
                for (int i = 0; i < PART; i += 8) st.put((p + i) / 8, v + i);
            }
            st.out((T *)a.out, first < 0 ? -1 : first + c, a.cols - c0 - c);
        }
    }
}

// The same for dh, val h and dval, from sums that the thread holds, of columns c0 to c0 + left (or W / 2).  The first part of h's rows is on its way to the stage.
template <typename T, int W>
__device__ __forceinline__ void take_held(const ProductArgs &a, const float (&held)[W / 2], const Stage<T, Shape<W>::TAKEN> &st, int64_t first, int64_t slot, int c0, int left,
                                          int part_of_sums, int64_t entry, float by)
{
    constexpr int PART = st.COLS;
    float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    st.fetched();
#pragma unroll
    for (int c = 0; c < W / 2; c += PART) {
        uint4 scaled[PART / 8], next[st.LANES];
#pragma unroll
        for (int i = 0; i < PART; i += 8) {
            float h[8], v[8];
            st.get(i / 8, h);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (entry >= 0) sum[j] = fmaf(held[c + i + j], h[j], sum[j]);
                v[j] = held[c + i + j] * by;
                h[j] *= by;                        // rounded to its type, as dz is, for the product with dy
            }
            Granule<T> packed;
            packed.pack(h);
            scaled[i / 8] = packed.w;
            st.put(i / 8, v);
        }
        st.out((T *)a.out, first < 0 ? -1 : first + c, left - c);
        const bool more = c + PART < W / 2;
        if (more) st.load(next, (const T *)a.other, first < 0 ? -1 : first + c + PART, left - c - PART);
        // a row of zeros adds nothing to the sums over an expert's tokens
#pragma unroll
        for (int i = 0; i < PART / 8; i++) st.at(st.lane, i) = scaled[i];
        st.out((T *)a.scaled, slot * a.cols + c0 + c, left - c);
        if (more) st.loaded(next);
    }
    if (entry >= 0) a.sums[part_of_sums * a.nnz + entry] = ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
}

// An entry whose column is no expert's: NaN.
template <typename T, int SUMS>
__device__ __forceinline__ void spoil(const ProductArgs &a, int thread)
{
    const int bad = SUMS == WEIGHT || SUMS == GATED_GRAD ? 0 : a.g.head[1];
    const float nan = __int_as_float(0x7fffffff);
    for (int i = blockIdx.x; i < bad; i += gridDim.x) {
        const int64_t entry = a.g.order[a.g.slots - 1 - i];
        for (int c = thread; c < a.cols; c += TAKERS) {
            if (SUMS == ENTRY_ROWS) a.sums[entry * a.cols + c] = nan;
            else ((T *)a.out)[entry * a.cols + c] = from_float<T>(nan);
        }
        if (SUMS == COMBINE_GRAD)
            for (int p = thread; p < 2 * a.tiles_n; p += TAKERS) a.sums[p * a.nnz + entry] = nan;
    }
}

// NUMBERED: the operand whose rows come by their number: A (the tile's rows), B (its columns, OUTER), or none
enum Numbered { NUMBERED_A, NUMBERED_B, NUMBERED_NONE };

template <typename T, int W, int FORM, int NUMBERED, int SUMS>
__global__ void __launch_bounds__(product_threads(W, SUMS), W == WIDE || segment(SUMS) ? 1 : 2)
product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const ProductArgs a)
{
    constexpr bool BF16 = !__is_same(T, __half);
    typedef Shape<W> S;
    constexpr int B_BYTES = S::B_BYTES, STEP_BYTES = S::STEP, RING = S::RING;
    constexpr unsigned TENSOR_BYTES = (NUMBERED == NUMBERED_A ? 0 : A_BYTES) + (NUMBERED == NUMBERED_B ? 0 : B_BYTES);
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) uint64_t bars[2 * RING + 4 + 1];
    __shared__ uint32_t tmem_room;
    __shared__ int broken_word;
    volatile int *broken = &broken_word;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int ISSUER = (TAKERS + FETCHERS) / 32, BOXES = ISSUER + 1, SEGMENT = segment(SUMS);
    const uint32_t ring = (smem_at(raw) + 1023) & ~1023u, full = smem_at(bars), empty = full + 8 * RING, done = empty + 8 * RING, taken = done + 16,
                   last = taken + 16;
    if (warp == ISSUER) tmem_alloc(smem_at(&tmem_room), 2 * W);
    if (tid == 0) {
        for (int i = 0; i < RING; i++) {
            bar_init(full + 8 * i, NUMBERED == NUMBERED_NONE ? 1 : 1 + FETCHERS);
            bar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; i++) {
            bar_init(done + 8 * i, 1);
            bar_init(taken + 8 * i, TAKERS / 32);
        }
        bar_init(last, 1);
        broken_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = tmem_room;
    wait_for_previous();

    const int mine = blockIdx.x, all = gridDim.x;
    // Tiles of a last round that would leave half of the CTAs idle are cut into two (dx of gated_grad_step 110 us, 114 with whole ones; v'dy of combine_grad_step, 3.3 rounds, gains 4, too).
    constexpr bool HALVES = W == WIDE && (SUMS == ENTRY_ROWS || SUMS == COMBINE_GRAD);
    const int entire = FORM == OUTER ? a.g.ngroups * a.tiles_m * a.tiles_n : a.g.head[0] * a.tiles_n;
    const int whole = HALVES && entire % all * 2 <= all ? entire / all * all : entire, tiles = whole + 2 * (entire - whole);
    auto tile_of = [&](int id) {
        Tile t;
        t.half = 0;
        if (HALVES && id >= whole) {
            t.half = 1 + (id - whole) % 2;
            id = whole + (id - whole) / 2;
        }
        if (FORM == OUTER) {
            t.group = id / (a.tiles_m * a.tiles_n);
            const int rest = id % (a.tiles_m * a.tiles_n);
            t.m = rest / a.tiles_n;
            t.n = rest % a.tiles_n;
            t.steps = (a.g.counts[t.group] + TK - 1) / TK;
            t.slot = a.g.first[t.group] * GROUP_TILE;
        } else {
            t.m = id / a.tiles_n;
            t.n = id % a.tiles_n;
            t.group = a.g.column[t.m];
            t.steps = (a.terms + TK - 1) / TK;
            t.slot = t.m * GROUP_TILE;
        }
        return t;
    };

    // what is under way lands before the CTA ends
    auto land = [&](unsigned step) {
        volatile int late = 0;
        for (unsigned i = step < RING ? 0 : step - RING; i < step; i++) bar_wait(full + 8 * (i % RING), i / RING & 1, &late);
    };
    if (warp >= TAKERS / 32) {
        if (many_registers(W, SUMS)) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == BOXES) {                           // fetches by tensor copies
            unsigned step = 0;                         // steps so far; stage = step % RING
            bool on = true;
            for (int id = mine; on && id < tiles; id += all) {
                const Tile t = tile_of(id);
                constexpr int BLOCKS = W / 64;
                const int n0 = t.n * W;
                for (int k = 0; k < t.steps; k++, step++) {
                    const unsigned s = step % RING;
                    const uint32_t to = ring + s * STEP_BYTES, bar = full + 8 * s;
                    on = __all_sync(0xffffffffu, bar_wait(empty + 8 * s, (step / RING & 1) ^ 1, broken));
                    if (!on) break;
                    if (elect()) {
                        bar_expect(bar, TENSOR_BYTES - (HALVES && t.half ? B_BYTES / 2 : 0));
                        if (HALVES && t.half) {
                            const int n = n0 + (t.half - 1) * (W / 2);
                            if (FORM == ROWS) {
                                load_box(to + A_BYTES, &map_b, k * TK, n, t.group, bar);
                            } else {
                                if (NUMBERED == NUMBERED_NONE) load_box(to, &map_a, k * TK, t.slot, 0, bar);
#pragma unroll
                                for (int i = 0; i < BLOCKS / 2; i++) load_box(to + A_BYTES + i * 8192, &map_b, n + i * 64, k * TK, t.group, bar);
                            }
                        } else if (FORM == ROWS) {
                            // an expert's gate rows, and as many up rows; or rows of the one weight
                            constexpr bool GATES = SUMS != ENTRY_ROWS;
                            load_box(to + A_BYTES, &map_b, k * TK, GATES ? t.n * (W / 2) : n0, GATES ? 2 * t.group : t.group, bar);
                            load_box(to + A_BYTES + B_BYTES / 2, &map_b, k * TK, GATES ? t.n * (W / 2) : n0 + W / 2, GATES ? 2 * t.group + 1 : t.group, bar);
                        } else if (FORM == BACK) {
                            if (NUMBERED == NUMBERED_NONE) load_box(to, &map_a, k * TK, t.slot, 0, bar);
#pragma unroll
                            for (int i = 0; i < BLOCKS; i++) load_box(to + A_BYTES + i * 8192, &map_b, n0 + i * 64, k * TK, t.group, bar);
                        } else if (NUMBERED == NUMBERED_A) {
#pragma unroll
                            for (int i = 0; i < BLOCKS; i++) load_box(to + A_BYTES + i * 8192, &map_b, n0 + i * 64, t.slot + k * TK, 0, bar);
                        } else {
#pragma unroll
                            for (int i = 0; i < 2; i++) load_box(to + i * 8192, &map_a, t.m * TM + i * 64, t.slot + k * TK, 0, bar);
                        }
                    }
                    __syncwarp();
                }
            }
            if (*broken) land(step);
        } else if (warp < ISSUER) {                    // fetches rows by their number
            unsigned step = 0;
            bool on = NUMBERED != NUMBERED_NONE;
            const int me = tid - TAKERS, chunk = me & 7, row = me >> 3;
            // a tile's row i is 128 bytes, of which chunk c lies at c ^ (i & 7): what tensor copies do, and the products undo
            const uint32_t at = row * 128 + ((chunk ^ (row & 7)) << 4);
            const char *base = (const char *)a.numbered + chunk * 16;
            const int64_t stride = a.ld * 2;
            for (int id = mine; on && id < tiles; id += all) {
                const Tile t = tile_of(id);
                const char *from[8];
                unsigned there = 0;
                if (NUMBERED == NUMBERED_A && FORM != OUTER) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int n = a.numbers[t.slot + row + 16 * i];
                        from[i] = base + max(n, 0) * stride;
                        there |= (n >= 0 ? 1u : 0u) << i;
                    }
                }
                int next[4];
                if (FORM == OUTER && t.steps)
#pragma unroll
                    for (int i = 0; i < 4; i++) next[i] = a.numbers[t.slot + row + 16 * i];
                for (int k = 0; k < t.steps; k++, step++) {
                    const unsigned s = step % RING;
                    const uint32_t to = ring + s * STEP_BYTES, bar = full + 8 * s;
                    on = __all_sync(0xffffffffu, bar_wait(empty + 8 * s, (step / RING & 1) ^ 1, broken));
                    if (!on) break;
                    if (FORM != OUTER) {
                        const bool in = k * TK + chunk * 8 < a.numbered_cols;
#pragma unroll
                        for (int i = 0; i < 8; i++) copy_or_zero(to + at + i * 2048, from[i] + (in ? k * TK * 2 : 0), in && (there >> i & 1));
                    } else {
                        constexpr int BLOCKS = NUMBERED == NUMBERED_A ? 2 : W / 64;
                        const uint32_t first = to + (NUMBERED == NUMBERED_A ? 0 : A_BYTES) + at;
                        const int col0 = NUMBERED == NUMBERED_A ? t.m * TM : t.n * W;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const char *src = base + max(next[i], 0) * stride;
#pragma unroll
                            for (int b = 0; b < BLOCKS; b++) {
                                const bool in = col0 + b * 64 + chunk * 8 < a.numbered_cols;
                                copy_or_zero(first + b * 8192 + i * 2048, src + (in ? (col0 + b * 64) * 2 : 0), in && next[i] >= 0);
                            }
                            if (k + 1 < t.steps) next[i] = a.numbers[t.slot + (k + 1) * TK + row + 16 * i];
                        }
                    }
                    copies_to(bar);
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else if (warp == ISSUER) {                   // issues the products
            // the whole warp goes along, and one thread of it issues: operands are the warp's then, not a thread's
            unsigned tile = 0, step = 0;
            bool on = true;
            int after = mine < tiles ? tile_of(mine).steps : 0;
            for (int id = mine; on && id < tiles; id += all) {
                const bool half = HALVES && id >= whole;
                const int steps = (int)__reduce_max_sync(0xffffffffu, (unsigned)after);  // the same in all, which the compiler does not know
                if (id + all < tiles) after = tile_of(id + all).steps;
                // steps from k0 to k1 of the tile, whose sums are taken out at once
                auto issue = [&](int k0, int k1) {
                    const unsigned b = tile & 1;
                    on = __all_sync(0xffffffffu, bar_wait(taken + 8 * b, (tile / 2 & 1) ^ 1, broken));
                    tmem_fence_after();
                    for (int k = k0; on && k < k1; k++, step++) {
                        const unsigned s = step % RING;
                        on = __all_sync(0xffffffffu, bar_wait(full + 8 * s, step / RING & 1, broken));
                        if (!on) break;
                        if (NUMBERED != NUMBERED_NONE) shared_to_products();
                        tmem_fence_after();
                        const uint32_t at = ring + s * STEP_BYTES;
                        const uint64_t da = tile_descriptor(at, 8192, 1024), db = tile_descriptor(at + A_BYTES, 8192, 1024);
                        // 16 terms: 32 bytes along a tile's rows, or 16 rows of 128 bytes
                        constexpr int next_a = FORM == OUTER ? 2048 / 16 : 32 / 16, next_b = FORM == ROWS ? 32 / 16 : 2048 / 16;
                        const uint32_t kind = half ? product_descriptor(BF16, TM, W / 2, FORM == OUTER, FORM != ROWS)
                                                   : product_descriptor(BF16, TM, W, FORM == OUTER, FORM != ROWS);
                        if (elect()) {
#pragma unroll
                            for (int i = 0; i < TK / 16; i++) product(tmem + b * W, da + i * next_a, db + i * next_b, kind, k - k0 + i > 0);
                            products_to(empty + 8 * s);
                            if (k + 1 == k1) products_to(done + 8 * b);
                        }
                        __syncwarp();
                    }
                    tile++;
                };
                if (steps == 0) continue;
                if constexpr (SEGMENT == 0) {
                    issue(0, steps);
                } else {
                    for (int k = 0; on && k < steps; k += SEGMENT) issue(k, min(k + SEGMENT, steps));
                }
            }
            if (*broken) {                             // products under way end before tensor memory is given back
                volatile int late = 0;
                if (elect()) products_to(last);
                bar_wait(last, 0, &late);
            }
            __syncwarp();
        }
    } else {                                       // takes the sums
        if (many_registers(W, SUMS)) asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
        spoil<T, SUMS>(a, tid);
        const int row = (warp & 3) * 32 + lane;
        unsigned char *room = raw + (ring - smem_at(raw)) + RING * STEP_BYTES + warp * 32 * S::TAKEN;
        unsigned tile = 0;
        for (int id = mine; id < tiles; id += all) {
            const Tile t = tile_of(id);
            const int64_t entry = FORM == OUTER ? -1 : a.g.order[t.slot + row];
            if constexpr (SEGMENT > 0) {
                const bool has = !t.half || warp < 4;
                const int half = t.half ? t.half - 1 : warp >> 2, c0 = t.n * W + half * (W / 2);
                const int64_t first = entry < 0 ? -1 : entry * a.cols + c0;
                const float by = entry >= 0 ? a.val[entry] : 0.0f;
                const Stage<T, S::TAKEN> st = {room, lane};
                if (has) st.fetch((const T *)a.other, first, a.cols - c0);
                float held[W / 2] = {};
                bool on = true;
                for (int k = 0; k < t.steps; k += SEGMENT, tile++) {
                    const unsigned b = tile & 1;
                    on = __all_sync(0xffffffffu, bar_wait(done + 8 * b, tile / 2 & 1, broken));
                    if (!on) break;
                    tmem_fence_after();
                    if (has) {
                        const uint32_t at = tmem + b * W + ((uint32_t)(warp & 3) << 21) + (t.half ? 0 : (warp >> 2) * (W / 2));
#pragma unroll
                        for (int c = 0; c < W / 2; c += 16) {
                            float v[16];
                            tmem_load(at + c, v);
#pragma unroll
                            for (int i = 0; i < 16; i++) held[c + i] += v[i];
                        }
                    }
                    tmem_fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(taken + 8 * b);
                }
                if (!on) break;
                if (has) take_held<T, W>(a, held, st, first, t.slot + row, c0, a.cols - c0, t.n * 2 + half, entry, by);
                continue;
            }
            const unsigned b = tile & 1;
            if (t.steps > 0) {
                if (!__all_sync(0xffffffffu, bar_wait(done + 8 * b, tile / 2 & 1, broken, t.steps))) break;
                tmem_fence_after();
            }
            const uint32_t at = tmem + b * W + ((uint32_t)(warp & 3) << 21);
            if (!HALVES || !t.half) take_sums<T, W, SUMS>(a, at, t.steps == 0, t, warp >> 2, row, entry, room);
            else if (warp < 4) take_sums<T, W, SUMS>(a, at - (t.half - 1) * (W / 2), false, t, t.half - 1, row, entry, room);
            if (t.steps > 0) {
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(taken + 8 * b);
                tile++;
            }
        }
        if (SEGMENT) asm volatile("cp.async.wait_all;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (warp == ISSUER) tmem_free(tmem, 2 * W);
    if (tid == 0 && *broken) a.g.head[2] = 1;
}

// A token's f32 rows, added in order: 8 columns a thread.
template <typename T>
__global__ void __launch_bounds__(256)
add_rows_kernel(int64_t nrows, int cols, const int64_t *__restrict__ pos, const float *__restrict__ sums, T *__restrict__ out)
{
    wait_for_previous();
    const int64_t parts = cols / 8, all = nrows * parts, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= all) return;
    const int64_t t = i / parts, c = i % parts * 8, lo = pos[t], hi = pos[t + 1];
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    const float4 *from = (const float4 *)(sums + lo * cols + c);
#pragma unroll 4
    for (int64_t e = lo; e < hi; e++, from += cols / 4) {
        const float4 x = __ldcs(from), y = __ldcs(from + 1);
        v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
        v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
    }
    store8<T>(out + t * cols + c, v);
}

__global__ void __launch_bounds__(256)
add_parts_kernel(int64_t n, int parts, const float *__restrict__ sums, float *__restrict__ out)
{
    wait_for_previous();
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float v = 0.0f;
    for (int p = 0; p < parts; p++) v += sums[p * n + i];
    out[i] = v;
}

// A single token: products of a weight's rows with its vectors, by the ordinary cores.  Neighbouring rows of an expert's weight are one piece of
// memory, so a CTA's share comes in copies of up to 32 KB.  Six teams of four warps have a stage each: while one of them works on its stage, the others'
// copies are under way, what an SM has to have in flight for the memory's full rate.  The vectors come through the L1 cache.
// 8 experts of 64, width 2048, inner 1024, gated and combine, us (and by the tensor cores): weights in L2 12.2 and 10.1 (16.6, 13.1), other experts' each time 16.5 and
// 11.8 (18.4, 14.5); with two tokens 32 and 18 (25, 14), so one is the limit.  2 of 8, 4096, 2048: 15.3 and 15.7 (22.8, 15.1); 4 of 32, 1024, 512: 4.7 and 4.7 (8.1, 7.7);
// 8 of 128, 2048, 768: 9.6 and 9.6 (16.6, 11.7); one of 16, 2048, 2048: 5.1 and 9.2 (13.0, 14.5); 8 of 64, 512, 256: 5.9 and 5.7 (5.7, 6.7).
// From memory, once in a while: 20.0 and 14.0 for the first; the copies alone 14.4 and 9.5 (67 and 34 MB, and 4 us of start-up).
static const int FEW_STAGES = 6, FEW_BYTES = 32 * 1024, FEW_SMEM = FEW_STAGES * FEW_BYTES, FEW_ENTRIES = 8, TEAM = 128, FEW_THREADS = FEW_STAGES * TEAM;

// Of R rows in shared memory, `next` bytes apart, and B vectors: a lane's part of their products.  A vector is loaded once for all the rows.
template <typename T, int R, int B>
__device__ __forceinline__ void dots(const unsigned char *row, unsigned next, const uint4 *const (&x)[B], int parts, int lane, float2 (&sum)[R][B])
{
    constexpr int N = Granule<T>::N;
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int i = 0; i < B; i++) sum[r][i] = make_float2(0.0f, 0.0f);
    constexpr int U = B == 1 ? 8 : 4;
    for (int c = lane; c < parts; c += 32 * U) {
        uint4 v[U][B];
#pragma unroll
        for (int j = 0; j < U; j++)
#pragma unroll
            for (int i = 0; i < B; i++) v[j][i] = c + 32 * j < parts ? __ldg(x[i] + c + 32 * j) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < U; j++)
            if (c + 32 * j < parts)
#pragma unroll
                for (int r = 0; r < R; r++) {
                    float2 w[N / 2];
                    Granule<T>{((const uint4 *)(row + r * next))[c + 32 * j]}.unpack(w);
#pragma unroll
                    for (int i = 0; i < B; i++) {
                        float2 y[N / 2];
                        Granule<T>{v[j][i]}.unpack(y);
#pragma unroll
                        for (int k = 0; k < N / 2; k++) sum[r][i] = fma2(w[k], y[k], sum[r][i]);
                    }
                }
    }
}

__device__ __forceinline__ void team_sync(int team) { asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(TEAM) : "memory"); }
// whether all threads of the team say so; a barrier of the team, too
__device__ __forceinline__ bool team_all(int team, bool v)
{
    unsigned all;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(all) : "r"((unsigned)v), "r"(team + 1), "n"(TEAM) : "memory");
    return all != 0;
}

// What both kernels do: steps, which the teams take in turn.  issue(step, stage's address, barrier) copies a step's rows, by one thread; prepare(step) looks up
// what else they are worked on with, while they are under way; take(stage) works on them.
template <typename Issue, typename Prepare, typename Take>
__device__ __forceinline__ void few_steps(int steps, unsigned char *ring, int *head, Issue issue, Prepare prepare, Take take)
{
    __shared__ __align__(8) uint64_t bars[FEW_STAGES];
    __shared__ int broken_word;
    volatile int *broken = &broken_word;
    const int team = threadIdx.x / TEAM;
    const bool first = threadIdx.x % TEAM == 0;
    unsigned char *stage = ring + team * FEW_BYTES;
    const uint32_t bar = smem_at(bars + team);
    if (threadIdx.x == 0) broken_word = 0;
    if (first) {
        bar_init(bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (team < steps) issue(team, smem_at(stage), bar);
    }
    __syncthreads();
    unsigned parity = 0;
    for (int step = team; step < steps; step += FEW_STAGES, parity ^= 1) {
        prepare(step);
        // A wait that runs out does so for the whole team: threads that went on alone would wait for the others at its next barrier.
        if (!team_all(team, bar_wait(bar, parity, broken))) {
            if (first) {                           // what is under way lands first
                volatile int late = 0;
                bar_wait(bar, parity, &late);
                head[2] = 1;
            }
            return;
        }
        take(stage);
        team_sync(team);
        if (first && step + FEW_STAGES < steps) issue(step + FEW_STAGES, smem_at(stage), bar);
    }
}

// Steps of `each` columns of h, gate and up rows of a tile's expert.
template <typename T>
__global__ void __launch_bounds__(FEW_THREADS)
gated_few_kernel(const ProductArgs a, const T *__restrict__ w, int each)
{
    extern __shared__ __align__(128) unsigned char ring[];
    wait_for_previous();
    const int lane = threadIdx.x & 31, warp = threadIdx.x % TEAM >> 5, inner = a.cols, width = a.terms, pieces = (inner + each - 1) / each;
    if (a.g.head[1] && threadIdx.x < TAKERS) spoil<T, GATED>(a, threadIdx.x);
    const int64_t units = (int64_t)a.g.head[0] * pieces;
    const int steps = units > blockIdx.x ? (int)((units - 1 - blockIdx.x) / gridDim.x) + 1 : 0;
    auto unit = [&](int step) { return blockIdx.x + (int64_t)step * gridDim.x; };
    const unsigned second = (unsigned)each * width * sizeof(T);
    int f = 0, slot = 0, count = 0, entry = 0;     // of the step: its first column, its tile's slots, entries, the first one's number and row
    const T *x0 = nullptr;
    few_steps(
        steps, ring, a.g.head,
        [&](int step, uint32_t to, uint32_t bar) {
            const int m = (int)(unit(step) / pieces), f = (int)(unit(step) % pieces) * each;
            const unsigned bytes = (unsigned)min(each, inner - f) * width * sizeof(T);
            const T *gate = w + ((int64_t)a.g.column[m] * 2 * inner + f) * width;
            bar_expect(bar, 2 * bytes);
            load_bytes(to, gate, bytes, bar);
            load_bytes(to + second, gate + (int64_t)inner * width, bytes, bar);
        },
        [&](int step) {
            const int m = (int)(unit(step) / pieces), group = a.g.column[m];
            f = (int)(unit(step) % pieces) * each;
            slot = m * GROUP_TILE;
            entry = a.g.order[slot];
            x0 = (const T *)a.numbered + a.numbers[slot] * a.ld;
            count = min(GROUP_TILE, a.g.counts[group] - (m - a.g.first[group]) * GROUP_TILE);
        },
        [&](const unsigned char *stage) {
            const int rows = min(each, inner - f), parts = width / 8;
            for (int r = warp; r < rows; r += TEAM / 32) {
                auto give = [&](auto batch, int e0) {
                    constexpr int B = decltype(batch)::value;
                    const uint4 *x[B];
#pragma unroll
                    for (int i = 0; i < B; i++) x[i] = (const uint4 *)(B == 1 && e0 == 0 ? x0 : (const T *)a.numbered + a.numbers[slot + e0 + i] * a.ld);
                    float2 sum[2][B];
                    dots<T, 2, B>(stage + (size_t)r * width * sizeof(T), second, x, parts, lane, sum);
#pragma unroll
                    for (int i = 0; i < B; i++) {
                        const float g = warp_sum(sum[0][i].x + sum[0][i].y), u = warp_sum(sum[1][i].x + sum[1][i].y);
                        if (lane == 0)
                            ((T *)a.out)[(int64_t)(B == 1 && e0 == 0 ? entry : a.g.order[slot + e0 + i]) * inner + f + r] = from_float<T>(g * logistic(gate_of(g, a.gelu).x) * u);
                    }
                };
                int e = 0;
                for (; e + 2 <= count; e += 2) give(std::integral_constant<int, 2>(), e);
                if (e < count) give(std::integral_constant<int, 1>(), e);
            }
        });
}

// Steps of `each` elements of a row of y: all its entries, eight at a time, two of them a warp; a team stays with its elements until they are summed.
template <typename T>
__global__ void __launch_bounds__(FEW_THREADS)
combine_few_kernel(const ProductArgs a, const int64_t *__restrict__ pos, const int64_t *__restrict__ crd, const T *__restrict__ v, int each)
{
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ float sums[FEW_STAGES][TEAM / 32][FEW_BYTES / FEW_ENTRIES / 16];      // a row has 16 bytes or more
    wait_for_previous();
    const int tid = threadIdx.x, lane = tid & 31, team = tid / TEAM, warp = tid % TEAM >> 5, width = a.rows, inner = a.terms;
    const int64_t first = pos[0], last = pos[1];
    // the CTA's pieces of y: blockIdx.x, + gridDim.x, ...; the team's: every FEW_STAGES-th of those, each in batches of eight entries
    const int pieces = (width + each - 1) / each, mine = pieces > (int)blockIdx.x ? (pieces - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0;
    const int batches = max(1, (int)((last - first + FEW_ENTRIES - 1) / FEW_ENTRIES)), count = mine > team ? (mine - 1 - team) / FEW_STAGES * batches + batches : 0;
    struct Step {
        int batch, d;
        int64_t lo, hi;
    };
    auto at = [&](int step) {
        const int n = step / FEW_STAGES, piece = (int)blockIdx.x + (team + n / batches * FEW_STAGES) * (int)gridDim.x;
        Step s = {n % batches, piece * each, 0, 0};
        s.lo = first + (int64_t)s.batch * FEW_ENTRIES;
        s.hi = min(s.lo + FEW_ENTRIES, last);
        return s;
    };
    const unsigned room = FEW_BYTES / FEW_ENTRIES;
    Step now = {0, 0, 0, 0};
    float by[FEW_ENTRIES / (TEAM / 32)] = {};      // the values of the warp's entries
    few_steps(
        count ? team + (count - 1) * FEW_STAGES + 1 : 0, ring, a.g.head,
        [&](int step, uint32_t to, uint32_t bar) {
            const Step s = at(step);
            const unsigned bytes = (unsigned)min(each, width - s.d) * inner * sizeof(T);
            bar_expect(bar, (unsigned)(s.hi - s.lo) * bytes);
            for (int64_t e = s.lo; e < s.hi; e++) {
                const int64_t col = crd[e];
                load_bytes(to + (unsigned)(e - s.lo) * room, v + ((col >= 0 && col < a.g.ngroups ? col : 0) * width + s.d) * inner, bytes, bar);
            }
        },
        [&](int step) {
            now = at(step);
#pragma unroll
            for (int i = 0; i < FEW_ENTRIES / (TEAM / 32); i++) {
                const int64_t e = now.lo + i * (TEAM / 32) + warp;
                if (e >= now.hi) break;
                const int64_t col = crd[e];
                by[i] = col >= 0 && col < a.g.ngroups ? a.val[e] : __int_as_float(0x7fffffff);
            }
        },
        [&](const unsigned char *stage) {
            const int rows = min(each, width - now.d);
            const unsigned next = (unsigned)inner * sizeof(T);
            auto give = [&](auto batch, int r) {
                constexpr int R = decltype(batch)::value;
                float sum[R] = {};
#pragma unroll
                for (int i = 0; i < FEW_ENTRIES; i += TEAM / 32) {
                    const int64_t e = now.lo + i + warp;
                    if (e >= now.hi) break;
                    const uint4 *const x[1] = {(const uint4 *)((const T *)a.numbered + e * inner)};
                    float2 d[R][1];
                    dots<T, R, 1>(stage + (i + warp) * room + r * next, next, x, inner / 8, lane, d);
#pragma unroll
                    for (int j = 0; j < R; j++) sum[j] = fmaf(by[i / (TEAM / 32)], d[j][0].x + d[j][0].y, sum[j]);
                }
#pragma unroll
                for (int j = 0; j < R; j++) {
                    const float s = warp_sum(sum[j]);
                    if (lane == 0) sums[team][warp][r + j] = now.batch == 0 ? s : sums[team][warp][r + j] + s;
                }
            };
            int r = 0;
            for (; r + 2 <= rows; r += 2) give(std::integral_constant<int, 2>(), r);
            if (r < rows) give(std::integral_constant<int, 1>(), r);
            if (now.hi < last) return;
            team_sync(team);
            for (int r = tid % TEAM; r < rows; r += TEAM)
                ((T *)a.out)[now.d + r] = from_float<T>((sums[team][0][r] + sums[team][1][r]) + (sums[team][2][r] + sums[team][3][r]));
        });
}

// Narrow tiles where wide ones would leave most SMs without any.  The number of tiles is on the device; its limit by the numbers of entries and experts decides.
// Gated products, us, wide and narrow: 16 to 40 wide tiles of 32 steps 16.7 and 13.4, 64 of them 16.8 and 17.2; 32 and 48 of 16 steps 10.9 and 8.5, 64 of them 10.9
// and 11.0, 145 11.1 and 15.6.  Sums of experts' outputs: 32 of 16 steps 12.5 and 10.4, 64 of them 12.7 and 12.8; 64 of 4 steps 8.1 and 7.5, 128 of them 8.4 and 10.4.
static bool narrow(const Groups &g, int64_t nnz, int64_t columns) { return (group_tiles(nnz, g.ngroups) - 1) * ceil_div(columns, WIDE) * 4 < sm_count(); }

template <typename T, int W, int FORM, int NUMBERED, int SUMS>
static int launch_product(const CUtensorMap &map_a, const CUtensorMap &map_b, ProductArgs a, int64_t columns, cudaStream_t st)
{
    typedef Shape<W> S;
    auto kernel = product_kernel<T, W, FORM, NUMBERED, SUMS>;
    CB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    a.tiles_n = (int)ceil_div(columns, W);
    if (FORM == OUTER) a.tiles_m = (int)ceil_div(a.rows, TM);
    const int64_t tiles = FORM == OUTER ? (int64_t)a.g.ngroups * a.tiles_m * a.tiles_n : (group_tiles(a.nnz, a.g.ngroups) - 1) * a.tiles_n;
    if (tiles > 0x3fffffffLL) return fail("experts: more than 2^30 tiles");
    const int64_t most = sm_count() * (W == WIDE ? 1 : 2);     // CTAs that run at the same time: each goes from tile to tile
    CB_CUDA(launch_behind(kernel, dim3((unsigned)(tiles < most ? tiles : most)), product_threads(W, SUMS), S::SMEM, st, map_a, map_b, a));
    return 0;
}

// The shape that a product of `columns` columns takes: wide tiles for sums over an expert's tokens; else narrow ones where wide ones are fewer than a quarter of the SMs.
template <typename T, int FORM, int NUMBERED, int SUMS, typename Maps>
static int launch_shape(const ProductArgs &a, int64_t columns, cudaStream_t st, Maps maps)
{
    alignas(64) CUtensorMap ma, mb;
    memset(&ma, 0, sizeof(ma));
    memset(&mb, 0, sizeof(mb));
    if constexpr (FORM == OUTER) {
        CB_TRY(maps(ma, mb, WIDE));
        return launch_product<T, WIDE, FORM, NUMBERED, SUMS>(ma, mb, a, columns, st);
    } else {
        if (narrow(a.g, a.nnz, columns)) {
            CB_TRY(maps(ma, mb, NARROW));
            return launch_product<T, NARROW, FORM, NUMBERED, SUMS>(ma, mb, a, columns, st);
        }
        CB_TRY(maps(ma, mb, WIDE));
        return launch_product<T, WIDE, FORM, NUMBERED, SUMS>(ma, mb, a, columns, st);
    }
}

struct Sizes {
    int64_t nrows, nexperts, nnz, width, inner;
};
static int check(const char *what, const Sizes &s)
{
    if (s.nrows < 0 || s.nnz < 0 || s.nexperts < 1 || s.nexperts > MOST_GROUPS)
        return fail("%s: %lld entries in %lld rows of %lld experts (1 to %d)", what, (long long)s.nnz, (long long)s.nrows, (long long)s.nexperts, MOST_GROUPS);
    if (s.nrows > 0x7ffffff0LL || s.nnz > 0x70000000LL) return fail("%s: more than 2^31 rows, or 1.8e9 entries", what);
    if (s.width < 8 || s.inner < 8 || s.width % 8 || s.inner % 8 || s.width > 1 << 20 || s.inner > 1 << 20)
        return fail("%s: width %lld and inner %lld; multiples of 8 up to 2^20", what, (long long)s.width, (long long)s.inner);
    return 0;
}
static int check_at(const char *what, const void *p)
{
    return (uintptr_t)p % 16 ? fail("%s: an address that is not a multiple of 16 bytes", what) : 0;
}
static int check_rows(const char *what, const void *p, int64_t ld, int64_t cols)
{
    if (ld < cols || ld % 8) return fail("%s: a row stride of %lld elements; a multiple of 8, and no less than the row's %lld", what, (long long)ld, (long long)cols);
    return check_at(what, p);
}

template <typename T>
static ProductArgs arguments(const Sizes &s, int32_t *plan)
{
    ProductArgs a;
    memset(&a, 0, sizeof(a));
    a.g = groups_in(plan, s.nnz, s.nexperts);
    a.nnz = s.nnz;
    return a;
}
template <typename T>
static constexpr bool is_bf16() { return !__is_same(T, __half); }

template <typename T>
static int add_rows(const Sizes &s, const int64_t *pos, const float *sums, void *out, cudaStream_t st)
{
    if (s.nrows == 0) return 0;
    CB_CUDA(launch_behind(add_rows_kernel<T>, dim3((unsigned)ceil_div(s.nrows * (s.width / 8), 256)), 256, 0, st, s.nrows, (int)s.width, pos, sums, (T *)out));
    return 0;
}

template <typename T>
static int gated_experts(const Sizes &s, int32_t gelu, int32_t *plan, const void *x, int64_t ldx, const void *w, void *h, cudaStream_t st)
{
    const char *what = "gated_experts";
    clear_error();
    CB_TRY(check(what, s));
    CB_TRY(check_rows(what, x, ldx, s.width));
    CB_TRY(check_at(what, w));
    CB_TRY(check_at(what, h));
    if (s.nnz == 0 || s.nrows == 0) return 0;
    ProductArgs a = arguments<T>(s, plan);
    a.number(a.g.token, x, ldx, s.width);
    a.terms = (int)s.width;
    a.cols = (int)s.inner;
    a.gelu = gelu != 0;
    a.out = h;
    if (s.nrows == 1 && s.width * 2 * (int64_t)sizeof(T) <= FEW_BYTES) {
        // no fewer steps than SMs, if there are rows enough
        const int64_t fit = FEW_BYTES / (s.width * 2 * (int64_t)sizeof(T)), most = group_tiles(s.nnz, s.nexperts) - 1, share = ceil_div(most * s.inner, sm_count());
        const int each = (int)(fit < share ? fit : share);
        const int64_t units = most * ceil_div(s.inner, each);
        CB_CUDA(cudaFuncSetAttribute(gated_few_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_SMEM));
        CB_CUDA(launch_behind(gated_few_kernel<T>, dim3((unsigned)(units < sm_count() ? units : sm_count())), FEW_THREADS, FEW_SMEM, st, a, (const T *)w, each));
        return 0;
    }
    return launch_shape<T, ROWS, NUMBERED_A, GATED>(a, 2 * s.inner, st, [&](CUtensorMap &, CUtensorMap &mb, int wide) {
        return make_box_map(what, w, is_bf16<T>(), 2 * s.nexperts, s.inner, s.width, wide / 2, &mb);
    });
}

// dz: room for slots x 2 inner; sums: for nnz x width floats (null with dx)
template <typename T>
static int gated_experts_grad(const Sizes &s, int32_t gelu, const int64_t *pos, int32_t *plan, const void *x, int64_t ldx, const void *w, const void *dh,
                              void *dz, float *sums, void *dx, void *dw, cudaStream_t st)
{
    const char *what = "gated_experts_grad";
    clear_error();
    CB_TRY(check(what, s));
    CB_TRY(check_rows(what, x, ldx, s.width));
    for (const void *p : {w, dh, (const void *)dz, (const void *)sums, (const void *)dx, (const void *)dw}) CB_TRY(check_at(what, p));
    if (s.nnz == 0 || s.nrows == 0) {
        if (dx) CB_CUDA(cudaMemsetAsync(dx, 0, s.nrows * s.width * sizeof(T), st));
        if (dw) CB_CUDA(cudaMemsetAsync(dw, 0, 2 * s.nexperts * s.inner * s.width * sizeof(T), st));
        return 0;
    }
    ProductArgs a = arguments<T>(s, plan);
    a.number(a.g.token, x, ldx, s.width);
    a.terms = (int)s.width;
    a.cols = (int)s.inner;
    a.gelu = gelu != 0;
    a.other = dh;
    a.out = dz;
    CB_TRY((launch_shape<T, ROWS, NUMBERED_A, GATED_GRAD>(a, 2 * s.inner, st, [&](CUtensorMap &, CUtensorMap &mb, int wide) {
        return make_box_map(what, w, is_bf16<T>(), 2 * s.nexperts, s.inner, s.width, wide / 2, &mb);
    })));
    if (dx) {
        a = arguments<T>(s, plan);
        a.terms = 2 * (int)s.inner;
        a.cols = (int)s.width;
        a.sums = sums;
        CB_TRY((launch_shape<T, BACK, NUMBERED_NONE, ENTRY_ROWS>(a, s.width, st, [&](CUtensorMap &mz, CUtensorMap &mb, int) {
            CB_TRY(make_box_map(what, dz, is_bf16<T>(), 1, a.g.slots, 2 * s.inner, TM, &mz));
            return make_box_map(what, w, is_bf16<T>(), s.nexperts, 2 * s.inner, s.width, TK, &mb);
        })));
        CB_TRY(add_rows<T>(s, pos, sums, dx, st));
    }
    if (dw) {
        a = arguments<T>(s, plan);
        a.number(a.g.token, x, ldx, s.width);
        a.rows = 2 * (int)s.inner;
        a.cols = (int)s.width;
        a.out = dw;
        CB_TRY((launch_shape<T, OUTER, NUMBERED_B, WEIGHT>(a, s.width, st, [&](CUtensorMap &mz, CUtensorMap &, int) {
            return make_box_map(what, dz, is_bf16<T>(), 1, a.g.slots, 2 * s.inner, TK, &mz);
        })));
    }
    return 0;
}

// sums: room for nnz x width floats
template <typename T>
static int combine_experts(const Sizes &s, const int64_t *pos, const int64_t *crd, int32_t *plan, const void *h, const float *val, const void *v, float *sums, void *y,
                           cudaStream_t st)
{
    const char *what = "combine_experts";
    clear_error();
    CB_TRY(check(what, s));
    for (const void *p : {h, v, (const void *)sums, (const void *)y}) CB_TRY(check_at(what, p));
    if (s.nnz == 0 || s.nrows == 0) {
        CB_CUDA(cudaMemsetAsync(y, 0, s.nrows * s.width * sizeof(T), st));
        return 0;
    }
    if (s.nrows == 1 && s.inner * (int64_t)sizeof(T) <= FEW_BYTES / FEW_ENTRIES) {
        const int64_t fit = FEW_BYTES / FEW_ENTRIES / (s.inner * (int64_t)sizeof(T)), share = ceil_div(s.width, sm_count());
        const int each = (int)(fit < share ? fit : share);
        const int64_t units = ceil_div(s.width, each);
        ProductArgs a = arguments<T>(s, plan);
        a.numbered = h;
        a.val = val;
        a.out = y;
        a.terms = (int)s.inner;
        a.rows = (int)s.width;
        CB_CUDA(cudaFuncSetAttribute(combine_few_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_SMEM));
        CB_CUDA(launch_behind(combine_few_kernel<T>, dim3((unsigned)(units < sm_count() ? units : sm_count())), FEW_THREADS, FEW_SMEM, st, a, pos, crd, (const T *)v, each));
        return 0;
    }
    ProductArgs a = arguments<T>(s, plan);
    a.number(a.g.order, h, s.inner, s.inner);
    a.terms = (int)s.inner;
    a.cols = (int)s.width;
    a.val = val;
    a.sums = sums;
    CB_TRY((launch_shape<T, ROWS, NUMBERED_A, ENTRY_ROWS>(a, s.width, st, [&](CUtensorMap &, CUtensorMap &mb, int wide) {
        return make_box_map(what, v, is_bf16<T>(), s.nexperts, s.width, s.inner, wide / 2, &mb);
    })));
    return add_rows<T>(s, pos, sums, y, st);
}

// scaled: room for slots x inner; sums: for nnz x 2 ceil(inner / 64) floats
template <typename T>
static int combine_experts_grad(const Sizes &s, int32_t *plan, const void *h, const float *val, const void *v, const void *dy, int64_t lddy, void *scaled,
                                float *sums, void *dh, void *dv, float *dval, cudaStream_t st)
{
    const char *what = "combine_experts_grad";
    clear_error();
    CB_TRY(check(what, s));
    CB_TRY(check_rows(what, dy, lddy, s.width));
    for (const void *p : {h, v, (const void *)scaled, (const void *)dh, (const void *)dv}) CB_TRY(check_at(what, p));
    if (s.nnz == 0 || s.nrows == 0) {
        if (dv) CB_CUDA(cudaMemsetAsync(dv, 0, s.nexperts * s.inner * s.width * sizeof(T), st));
        return 0;
    }
    ProductArgs a = arguments<T>(s, plan);
    a.number(a.g.token, dy, lddy, s.width);
    a.terms = (int)s.width;
    a.cols = (int)s.inner;
    a.other = h;
    a.val = val;
    a.out = dh;
    a.scaled = scaled;
    a.sums = sums;
    int parts = 0;
    CB_TRY((launch_shape<T, BACK, NUMBERED_A, COMBINE_GRAD>(a, s.inner, st, [&](CUtensorMap &, CUtensorMap &mb, int wide) {
        parts = 2 * (int)ceil_div(s.inner, wide);
        return make_box_map(what, v, is_bf16<T>(), s.nexperts, s.width, s.inner, TK, &mb);
    })));
    CB_CUDA(launch_behind(add_parts_kernel, dim3((unsigned)ceil_div(s.nnz, 256)), 256, 0, st, s.nnz, parts, sums, dval));
    if (dv) {
        a = arguments<T>(s, plan);
        a.number(a.g.token, dy, lddy, s.width);
        a.rows = (int)s.width;
        a.cols = (int)s.inner;
        a.out = dv;
        CB_TRY((launch_shape<T, OUTER, NUMBERED_A, WEIGHT>(a, s.inner, st, [&](CUtensorMap &, CUtensorMap &mh, int) {
            return make_box_map(what, scaled, is_bf16<T>(), 1, a.g.slots, s.inner, TK, &mh);
        })));
    }
    return 0;
}

}  // namespace cb200

#define EXPERTS(suffix, T)                                                                                                                             \
    extern "C" int32_t comet_b200_dev_gated_experts_##suffix##_i64(int64_t nrows, int64_t nexperts, int64_t nnz, int64_t width, int64_t inner,         \
                                                                   int32_t gelu, int32_t *plan, const void *x, int64_t ldx, const void *w, void *h,     \
                                                                   void *stream)                                                                       \
    {                                                                                                                                                  \
        return cb200::gated_experts<T>({nrows, nexperts, nnz, width, inner}, gelu, plan, x, ldx, w, h, (cudaStream_t)stream);                          \
    }                                                                                                                                                  \
    extern "C" int32_t comet_b200_dev_gated_experts_grad_##suffix##_i64(                                                                               \
        int64_t nrows, int64_t nexperts, int64_t nnz, int64_t width, int64_t inner, int32_t gelu, const int64_t *pos, int32_t *plan, const void *x,     \
        int64_t ldx, const void *w, const void *dh, void *dz, float *sums, void *dx, void *dw, void *stream)                                           \
    {                                                                                                                                                  \
        return cb200::gated_experts_grad<T>({nrows, nexperts, nnz, width, inner}, gelu, pos, plan, x, ldx, w, dh, dz, sums, dx, dw,                    \
                                            (cudaStream_t)stream);                                                                                     \
    }                                                                                                                                                  \
    extern "C" int32_t comet_b200_dev_combine_experts_##suffix##_i64(int64_t nrows, int64_t nexperts, int64_t nnz, int64_t width, int64_t inner,       \
                                                                     const int64_t *pos, const int64_t *crd, int32_t *plan, const void *h, const float *val, \
                                                                     const void *v, float *sums, void *y, void *stream)                                \
    {                                                                                                                                                  \
        return cb200::combine_experts<T>({nrows, nexperts, nnz, width, inner}, pos, crd, plan, h, val, v, sums, y, (cudaStream_t)stream);                   \
    }                                                                                                                                                  \
    extern "C" int32_t comet_b200_dev_combine_experts_grad_##suffix##_i64(                                                                             \
        int64_t nrows, int64_t nexperts, int64_t nnz, int64_t width, int64_t inner, int32_t *plan, const void *h, const float *val, const void *v,      \
        const void *dy, int64_t lddy, void *scaled, float *sums, void *dh, void *dv, float *dval, void *stream)                                        \
    {                                                                                                                                                  \
        return cb200::combine_experts_grad<T>({nrows, nexperts, nnz, width, inner}, plan, h, val, v, dy, lddy, scaled, sums, dh, dv, dval,             \
                                              (cudaStream_t)stream);                                                                                   \
    }
EXPERTS(bf16, __nv_bfloat16)
EXPERTS(f16, __half)
