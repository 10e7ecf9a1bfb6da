// Entries of a CSR matrix grouped by column: a stable counting sort in one launch, by a cluster of up to sixteen CTAs.
//
// A warp has a stretch of rows and counts their entries by column (lanes with the same column find each other by votes on its bits, so there
// are no atomics and the order is always the same), the counts are summed over the warps and, through the
// cluster's shared memory, over the CTAs, and a second walk over the rows puts each entry where the sums say.
//
// Bound: instructions of the walks (votes, the search for a row), and the chains of loads and sums around them: 8192 rows of 8 among 64 columns 20 us, 777 rows 12, one row 5.
#include <atomic>
#include <type_traits>

#include "groups.cuh"
#include "logits.cuh"
#include "stream.cuh"

namespace cb200 {

static const int GT = 1024, GW = GT / 32;
// entries of a CTA that its shared memory has room for beside the counts
__host__ __device__ inline int most_sorted(int ngroups) { return ngroups <= 512 ? 8192 : 4096; }
static size_t room_for(int64_t ngroups) { return (size_t)ngroups * GW * sizeof(int) + most_sorted((int)ngroups) * (sizeof(int2) + sizeof(short)); }

__global__ void __launch_bounds__(GT)
group_kernel(int64_t nrows, int64_t nnz, const int64_t *__restrict__ pos, const int64_t *__restrict__ crd, const Groups g)
{
    extern __shared__ __align__(16) int warps[];   // [GW][ngroups]: a warp's entries of a column, then the slot of its next one
    __shared__ int mine[MOST_GROUPS], start[MOST_GROUPS], whole[MOST_GROUPS], ends[MOST_GROUPS], local[MOST_GROUPS], sums[GW + 1];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = g.ngroups;
    const unsigned rank = cluster_rank(), ranks = cluster_size();
    int *own = warps + (size_t)warp * n;
    let_next_start();                              // it waits for this one's end before it reads
    wait_for_previous();
    for (int i = tid; i < GW * n; i += GT) warps[i] = 0;
    if (rank == 0 && tid < GROUP_HEAD) g.head[tid] = 0;
    __syncthreads();
    const int64_t each = (nrows + (int64_t)ranks * GW - 1) / ((int64_t)ranks * GW), from = min((rank * GW + warp) * each, nrows);
    const int64_t to = min(from + each, nrows);
    const int bits = 32 - __clz(n - 1);            // of a column (a vote a bit: match.any takes some 200 clocks, 6 votes 40)
    // The entries of 32 rows after the other, a lane an entry, four loads on their way at a time; what(entry, its row, its column, the lanes that have the
    // same one, whether there is one) by all lanes.  ROWS: the row is asked for, too; lane i knows where row r + i ends.
    auto walk = [&](auto rows, auto what) {
        for (int64_t r = from; r < to; r += 32) {
            const int64_t end = min(max(pos[min(r + lane + 1, to)], (int64_t)0), nnz), begin = min(max(pos[r], (int64_t)0), nnz);
            const int64_t hi = __shfl_sync(0xffffffffu, end, 31);
            const int ends_at = (int)(end - begin);
            for (int64_t e0 = begin; e0 < hi; e0 += 128) {
                int64_t col[4];
#pragma unroll
                for (int i = 0; i < 4; i++) col[i] = e0 + 32 * i + lane < hi ? crd[e0 + 32 * i + lane] : -1;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int64_t e = e0 + 32 * i + lane;
                    if (e0 + 32 * i >= hi) break;
                    const int c = col[i] >= 0 && col[i] < n ? (int)col[i] : -1;
                    unsigned alike = __ballot_sync(0xffffffffu, c >= 0);
#pragma unroll
                    for (int b = 0; b < 10; b++) {
                        if (b >= bits) break;
                        const bool set = c & 1 << b;
                        alike &= __ballot_sync(0xffffffffu, set) ^ (set ? 0u : ~0u);
                    }
                    int row = 0;                   // the first one that ends behind the entry
                    if (decltype(rows)::value)
#pragma unroll
                        for (int step = 16; step > 0; step /= 2) row += __shfl_sync(0xffffffffu, ends_at, row + step - 1) <= (int)(e - begin) ? step : 0;
                    what(e, r + row, c, alike, e < hi);
                    __syncwarp();
                }
            }
        }
    };
    walk(std::false_type(), [&](int64_t, int64_t, int col, unsigned alike, bool) {
        if (col >= 0 && lane == __ffs(alike) - 1) own[col] += __popc(alike);
    });
    __syncthreads();
    int total = 0, before = 0;
    if (tid < n) {
        int sum = 0;
        for (int w = 0; w < GW; w++) {
            const int v = warps[w * n + tid];
            warps[w * n + tid] = sum;
            sum += v;
        }
        mine[tid] = sum;
    }
    __syncthreads();
    if (ranks > 1) {
        cluster_arrive();
        cluster_wait();
    }
    if (tid < n)
        for (unsigned r = 0; r < ranks; r++) {
            const int v = ranks > 1 ? peer_load(&mine[tid], r) : mine[tid];
            if (r < rank) before += v;
            total += v;
        }
    // the CTA's own, one column after the other
    {
        int v = tid < n ? mine[tid] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int w = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += w;
        }
        if (lane == 31) sums[warp] = v;
        __syncthreads();
        for (int w = 0; w < warp; w++) v += sums[w];
        if (tid < n) local[tid] = v - mine[tid];
        __syncthreads();
        if (tid == GT - 1) sums[GW] = v;
    }
    const int tiles = (total + GROUP_TILE - 1) / GROUP_TILE;
    int upto = tiles;                              // inclusive sums over the columns
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    for (int w = 0; w < warp; w++) upto += sums[w];
    if (tid < n) {
        start[tid] = (upto - tiles) * GROUP_TILE + before;
        whole[tid] = total;
        ends[tid] = upto;
        if (rank == 0) {
            g.counts[tid] = total;
            g.first[tid] = upto - tiles;
            if (tid == n - 1) g.first[n] = g.head[0] = upto;
        }
    }
    __syncthreads();
    for (int c = rank * GW + warp; c < n; c += ranks * GW) {                         // a warp has a column's tiles and the rest of its last one
        const int sum = whole[c], first = ends[c] - (sum + GROUP_TILE - 1) / GROUP_TILE;
        for (int i = first + lane; i < ends[c]; i += 32) g.column[i] = c;
        for (int64_t i = (int64_t)first * GROUP_TILE + sum + lane; i < (int64_t)ends[c] * GROUP_TILE; i += 32) g.order[i] = g.token[i] = -1;
    }
    // where a warp's entries go: to their slots, or to their places among the CTA's own
    const int here = sums[GW], sortable = most_sorted(n);
    for (int i = tid; i < GW * n; i += GT) warps[i] += here <= sortable ? local[i % n] : start[i % n];
    __syncthreads();
    if (here <= sortable)
        for (int c = tid; c < n; c += GT) start[c] -= local[c];
    if (ranks > 1) cluster_arrive();               // this CTA has read the others' counts
    // Few enough for shared memory: the CTA's entries are put in order there, and leave in runs (a column's are next to each other).
    int2 *sorted = (int2 *)(warps + (size_t)GW * n);
    unsigned short *of = (unsigned short *)(sorted + sortable);
    const bool staged = here <= sortable;
    walk(std::true_type(), [&](int64_t e, int64_t row, int col, unsigned alike, bool on) {
        const int at = col >= 0 ? own[col] + __popc(alike & ((1u << lane) - 1)) : 0;
        __syncwarp();                              // all lanes at once: a wait for those alike would be one after the other
        if (col >= 0) {
            if (lane == 31 - __clz(alike)) own[col] = at + 1;
            if (staged) {
                sorted[at] = make_int2((int)e, (int)row);
                of[at] = (unsigned short)col;
            } else {
                g.order[at] = (int)e;
                g.token[at] = (int)row;
            }
        } else if (on) {
            g.order[g.slots - 1 - atomicAdd(&g.head[1], 1)] = (int)e;
        }
    });
    if (staged) {
        __syncthreads();
        for (int i = tid; i < here; i += GT) {
            const int2 v = sorted[i];
            const int at = start[of[i]] + i;
            g.order[at] = v.x;
            g.token[at] = v.y;
        }
    }
    __syncwarp();
    if (ranks > 1) cluster_wait();                 // its own stay until they have been read
}

// The same for few entries of few rows: a thread has an entry, and counts those of its column before it.
static const int FEW = 256, FEW_ROWS = 1024;
__global__ void __launch_bounds__(FEW)
group_few_kernel(int nrows, int nnz, const int64_t *__restrict__ pos, const int64_t *__restrict__ crd, const Groups g)
{
    __shared__ int rows[FEW_ROWS + 1], cols[FEW], count[MOST_GROUPS], first[MOST_GROUPS], sums[FEW / 32], bad;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = g.ngroups;
    let_next_start();
    wait_for_previous();
    const int64_t mine = tid < nnz ? crd[tid] : -1;
    for (int i = tid; i <= nrows; i += FEW) rows[i] = (int)min(max(pos[i], (int64_t)0), (int64_t)nnz);
    int col = mine >= 0 && mine < n ? (int)mine : -1;
    for (int i = tid; i < n; i += FEW) count[i] = 0;
    if (tid == 0) bad = 0;
    __syncthreads();
    const bool there = tid >= rows[0] && tid < rows[nrows];    // pos may be that of some rows of a larger matrix: the other rows' entries are none here
    if (!there) col = -1;
    cols[tid] = col;
    __syncthreads();
    int before = 0, row = 0;
    if (there) {
        if (col >= 0) atomicAdd(&count[col], 1);
        for (int i = 0; i < tid; i++) before += cols[i] == col;
        for (int step = FEW_ROWS / 2; step > 0; step /= 2)                           // the last row that begins at or before the entry
            if (row + step < nrows && rows[row + step] <= tid) row += step;
    }
    __syncthreads();
    // each thread: four columns
    int tiles = 0, upto;
    for (int i = 4 * tid; i < min(4 * tid + 4, n); i++) tiles += (count[i] + GROUP_TILE - 1) / GROUP_TILE;
    upto = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    for (int w = 0; w < warp; w++) upto += sums[w];
    int at = upto - tiles;
    for (int i = 4 * tid; i < min(4 * tid + 4, n); i++) {
        first[i] = at;
        g.first[i] = at;
        g.counts[i] = count[i];
        for (int e = 0; e < count[i]; e += GROUP_TILE) g.column[at++] = i;
    }
    if (tid == FEW - 1) g.first[n] = upto;
    if (tid > 0 && tid < GROUP_HEAD && tid != 1) g.head[tid] = 0;
    if (tid == FEW - 1) g.head[0] = upto;
    __syncthreads();
    for (int c = warp; c < n; c += FEW / 32) {
        const int sum = count[c], end = (sum + GROUP_TILE - 1) / GROUP_TILE * GROUP_TILE;
        for (int i = sum + lane; i < end; i += 32) g.order[first[c] * GROUP_TILE + i] = g.token[first[c] * GROUP_TILE + i] = -1;
    }
    if (there) {
        if (col >= 0) {
            g.order[first[col] * GROUP_TILE + before] = tid;
            g.token[first[col] * GROUP_TILE + before] = row;
        } else {
            g.order[g.slots - 1 - atomicAdd(&bad, 1)] = tid;
        }
    }
    __syncthreads();
    if (tid == 0) g.head[1] = bad;
}

static int group_entries(int64_t nrows, int64_t ncols, int64_t nnz, const int64_t *pos, const int64_t *crd, int32_t *plan, cudaStream_t st)
{
    clear_error();
    if (nrows < 0 || nnz < 0 || ncols < 1 || ncols > MOST_GROUPS)
        return fail("group_entries: %lld entries in %lld rows of %lld columns (1 to %d)", (long long)nnz, (long long)nrows, (long long)ncols, MOST_GROUPS);
    if (nrows > 0x7fffffffLL || nnz > 0x70000000LL) return fail("group_entries: more than 2^31 rows, or 1.8e9 entries");
    // one token's 8 entries: 4.9 us, 7.1 by the cluster's kernel
    if (nnz <= FEW && nrows <= FEW_ROWS) {
        CB_CUDA(launch_behind(group_few_kernel, dim3(1), FEW, 0, st, (int)nrows, (int)nnz, pos, crd, groups_in(plan, nnz, ncols)));
        return 0;
    }
    static std::atomic<int> most_ranks[64];        // of a device: 16, if it has room for a cluster of so many, else what every device takes
    int device = 0;
    CB_CUDA(cudaGetDevice(&device));
    // the limit of shared memory is that of the largest call, in every call
    CB_CUDA(cudaFuncSetAttribute(group_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)room_for(MOST_GROUPS)));
    CB_CUDA(cudaFuncSetAttribute(group_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(GT);
    cfg.dynamicSmemBytes = room_for(MOST_GROUPS);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    int most = device < 64 ? most_ranks[device].load() : MOST_CLUSTER;
    if (!most) {
        cfg.gridDim = dim3(16);
        attr[1].val.clusterDim.x = 16;
        int clusters = 0;
        most = cudaOccupancyMaxActiveClusters(&clusters, group_kernel, &cfg) == cudaSuccess && clusters > 0 ? 16 : MOST_CLUSTER;
        cudaGetLastError();                        // a refusal is an answer
        most_ranks[device].store(most);
    }
    // A share of 256 rows and more clusters pay, 8 entries a row, us: 777 rows 12 by four CTAs, 19 by one; 4096 rows 13 by 16, 22 by four; 8192 rows 20 by 16, 27 by
    // eight.
    int ranks = 1;
    while (ranks < most && nrows > (int64_t)ranks * GT / 4) ranks *= 2;
    cfg.gridDim = dim3((unsigned)ranks);
    attr[1].val.clusterDim.x = ranks;
    cfg.dynamicSmemBytes = room_for(ncols);
    CB_CUDA(cudaLaunchKernelEx(&cfg, group_kernel, nrows, nnz, pos, crd, groups_in(plan, nnz, ncols)));
    return 0;
}

}  // namespace cb200

extern "C" int64_t comet_b200_dev_group_entries_size(int64_t nnz, int64_t ncols) { return cb200::group_size(nnz, ncols); }

extern "C" int32_t comet_b200_dev_group_entries_i64(int64_t nrows, int64_t ncols, int64_t nnz, const int64_t *pos, const int64_t *crd, int32_t *plan,
                                                    void *stream)
{
    return cb200::group_entries(nrows, ncols, nnz, pos, crd, plan, (cudaStream_t)stream);
}
