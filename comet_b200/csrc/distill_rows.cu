// The distillation loss (distill.cu has the mathematics) of a batch that fills the chip: a CTA takes a row at a time.
//
// A row is cut into chunks of four granules (16 bytes) a thread, which go through a ring of six slots a thread in shared memory: a thread
// copies, reads and overwrites only slots of its own, and as soon as it has read one for the last time the next chunk's copy goes there.
// The first pass leaves a row's last six chunks in the ring; the second takes those, then has the first ones copied again (from L2,
// where a row has more than six: 48, 96 and 192 KB with CTAs of 128, 256 and 512 threads), and the next row's copies follow.
//
// The entries are taken by threads of their own, one each, ahead of time like the row (their columns and values two rows ahead, the 16
// bytes of X that each lies in one row): a bitmap marks the granules that hold some, the passes leave those out, and the thread of a
// granule's first entry takes it.  So the gradient is written once, no thread looks for entries, and a row has two barriers.
#include "distill.cuh"

namespace cb200 {

static const int BATCH = 4, SLOTS = 6;             // granules of a thread in a chunk; chunks in shared memory

__global__ void __launch_bounds__(1024)
distill_sum_kernel(const DistillArgs a)
{
    __shared__ double room[32];
    wait_for_previous();
    add_rows<1024>(a, room);
}

// Waits until no more than `n` of the thread's groups of copies are on their way.
__device__ __forceinline__ void wait_copies_but(int n)
{
    switch (n) {
    case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
    case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
    case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
    case 3: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
    case 4: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
    case 5: asm volatile("cp.async.wait_group 5;" ::: "memory"); break;
    default: asm volatile("cp.async.wait_group 6;" ::: "memory"); break;
    }
}

// A thread's elements so far: their maximum, and sums of 2^((x - maximum) c).
struct Sums {
    Exponent u;
    float m, stored;
    float2 s;
    __device__ __forceinline__ Sums(float c) : u(MINUS_INF, c), m(MINUS_INF), stored(0.0f), s(make_float2(0.0f, 0.0f)) {}
    __device__ __forceinline__ void raise(float most)
    {
        const float nm = max_nan(m, most);
        if (nm != m) {
            const Exponent to(nm, u.c);
            const float f = m == MINUS_INF ? 0.0f : exp2_fast(u.to(to));
            s = mul2(s, make_float2(f, f));
            stored *= f;
            m = nm;
            u = to;
        }
    }
    template <typename T>
    __device__ __forceinline__ void add_near(const Granule<T> &g)
    {
        constexpr int N = Granule<T>::N;
        float2 v[N / 2];
        g.unpack(v);
#pragma unroll
        for (int k = 0; k < N / 2; k++) {
            v[k] = u.of(v[k]);
            s = add2(s, make_float2(exp2_fast(v[k].x), exp2_fast(v[k].y)));
        }
    }
    template <typename T>
    __device__ __forceinline__ void add_any(const Granule<T> &g)
    {
        constexpr int N = Granule<T>::N;
        float v[N];
        g.unpack(v);
#pragma unroll
        for (int k = 0; k < N; k++) s.x += exp2_fast(u.of(v[k]));
    }
};

// A row's entries as a warp has seen them: the largest z and x, and with p' = 2^((z - reference) c) the sums of p', p' (z - reference) c
// and p' (x - largest x) c.  The reference is lse, or the largest z.  And the row's elements: their maximum, and sums of
// 2^((x - maximum) c) where nothing is stored and where something is.
struct Seen {
    float z, x, p, plogp, pu, m, others, stored;
};

// A row's entries' bounds, its weight, and lse.
struct Row {
    int64_t lo;
    int n;                                         // 0 too if the weight is
    float w, lse;
    __device__ __forceinline__ Row(const DistillArgs &a, int64_t t) : lo(0), n(0), w(0.0f), lse(0.0f)
    {
        if (t < a.nrows) {
            lo = a.pos[t];
            const int64_t many = a.pos[t + 1] - lo;
            w = a.weight ? a.weight[t] : 1.0f;
            if (a.lse) lse = a.lse[t];
            n = w != 0.0f ? (int)min(max(many, (int64_t)0), (int64_t)0x7fffffff) : 0;
        }
    }
};

// The first MANY entries of three rows on their way and in use; thread i's are the i-th.
template <typename TV, int MANY>
struct Staged {
    int64_t col[3][MANY];
    TV z[3][MANY];
    int prev[3][MANY];                             // the column before, as far as it is a column
    uint4 granule[2][MANY];
};

// 16 bytes, from and to BYTES behind the addresses
template <int BYTES>
__device__ __forceinline__ void copy_far(uint32_t to, const void *from)
{
    asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %2], 16;" ::"r"(to), "l"(from), "n"(BYTES) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void copy_small(void *to, const void *from)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "n"(BYTES) : "memory");
}

// Where a row of X lies: its granules, and elements before it in the first one.
template <typename T>
struct Place {
    const T *x;
    const uint4 *from;
    int off, all;
    __device__ __forceinline__ Place(const DistillArgs &a, int64_t t)
    {
        x = (const T *)a.x + t * a.ldx;
        from = (const uint4 *)((uintptr_t)x & ~(uintptr_t)15);
        off = (int)((uintptr_t)x & 15) / (int)sizeof(T);
        all = (off + a.ncols + Granule<T>::N - 1) / Granule<T>::N;
    }
    __device__ __forceinline__ int granule_of(int64_t col) const { return (int)(off + col) / Granule<T>::N; }
    // granule i, -inf where there is no row
    __device__ __forceinline__ Granule<T> masked(uint4 w, int i, int ncols) const
    {
        Granule<T> g;
        g.w = w;
        T *v = (T *)&g.w;
#pragma unroll
        for (int k = 0; k < Granule<T>::N; k++) {
            const int col = i * Granule<T>::N + k - off;
            if (col < 0 || col >= ncols) v[k] = from_float<T>(MINUS_INF);
        }
        return g;
    }
};

template <typename T, typename TV, int THREADS, bool REST, bool GRAD>
__global__ void __launch_bounds__(THREADS, 512 / THREADS)
distill_rows_kernel(const DistillArgs a, const int chunks, const int ring)
{
    constexpr int N = Granule<T>::N, WARPS = THREADS / 32, CHUNK = BATCH * THREADS, MANY = THREADS / 2;
    extern __shared__ uint4 slots[];               // ring * CHUNK; behind them, twice, a bit per granule: a thread of its own takes it
    __shared__ Seen seen[2][WARPS];
    __shared__ Staged<TV, MANY> staged;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int words = chunks * (CHUNK / 32);
    uint32_t *taken_twice = (uint32_t *)(slots + ring * CHUNK);
    const int again = GRAD ? chunks - ring : 0;       // a row's first chunks that are copied twice
    const int mine0 = warp * (BATCH * 32) + lane;  // the thread's granules of a chunk: this one and three more, 32 apart

    // The chunks in the order in which they go through the ring: a row's, its first ones again, the next row's.
    const uint32_t ring_begin = (uint32_t)__cvta_generic_to_shared(slots + mine0), ring_end = ring_begin + ring * (CHUNK * 16);
    uint32_t put = ring_begin;                     // slot of the next copy
    const Granule<T> *const use_begin = (const Granule<T> *)slots + mine0, *const use_end = use_begin + ring * CHUNK;
    const Granule<T> *use = use_begin;             // and of the next use
    const uint4 *source = nullptr;
    int to_come = 0, left = 0;                     // copies of the row still to be asked for; granules from this one on
    bool twice = false;                            // the row's first ones have been asked for a second time
    auto copy_row = [&](const Place<T> &r, bool reads, int many) {
        source = r.from + mine0;
        left = reads ? r.all - mine0 : 0;
        to_come = many;
    };
    // `here` is the row that is copied, `there` the one after it
    auto copy_next = [&](const Place<T> &here, bool reads, const Place<T> &there, bool there_reads) {
        if (to_come == 0) {
            twice = !twice && again > 0;
            if (twice) copy_row(here, reads, again);
            else copy_row(there, there_reads, chunks);
        }
        if (left > 3 * 32) {
            copy_far<0>(put, source);
            copy_far<512>(put, source);
            copy_far<1024>(put, source);
            copy_far<1536>(put, source);
        } else {
            if (left > 0) copy_far<0>(put, source);
            if (left > 32) copy_far<512>(put, source);
            if (left > 64) copy_far<1024>(put, source);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        put += CHUNK * 16;
        if (put == ring_end) put = ring_begin;
        source += CHUNK;
        left -= CHUNK;
        to_come--;
    };
    auto copy_entries = [&](const Row &r, int third) {
        if (tid < MANY && tid < r.n) {
            copy_small<8>(&staged.col[third][tid], a.crd + r.lo + tid);
            copy_small<sizeof(TV)>(&staged.z[third][tid], (const TV *)a.val + r.lo + tid);
            if (tid > 0) copy_small<4>(&staged.prev[third][tid], a.crd + r.lo + tid - 1);
        }
    };
    auto copy_entry_granules = [&](const Row &r, int third, int turn, const Place<T> &at) {
        if (tid < MANY && tid < r.n) {
            const int64_t col = staged.col[third][tid];
            if (col >= 0 && col < a.ncols) copy_granule(&staged.granule[turn][tid], at.from + at.granule_of(col));
        }
    };
    // the first or the last entry's column, for the two threads that may have to take an edge of the row
    auto end_of = [&](const Row &r) {
        if (r.n > 0 && tid >= THREADS - 2) return a.crd[tid == THREADS - 1 ? r.lo : r.lo + r.n - 1];
        return (int64_t)-1;
    };

    int64_t t = blockIdx.x;
    const int64_t step = gridDim.x;
    Row now(a, t), next(a, t + step), later(a, t + 2 * step);
    int64_t end = end_of(now);
    copy_entries(now, 0);
    copy_entries(next, 1);
    for (int i = tid; i < 2 * words; i += THREADS) taken_twice[i] = 0;
    wait_copies();
    {
        const Place<T> here(a, t), there(a, t + step);
        copy_entry_granules(now, 0, 0, here);
        asm volatile("cp.async.commit_group;" ::: "memory");
        copy_row(here, now.n > 0, chunks);
        for (int c = 0; c < ring; c++) copy_next(here, now.n > 0, there, next.n > 0);
    }
    __syncthreads();

    int third = 0;
    for (int turn = 0; t < a.nrows; t += step, turn ^= 1, third = third == 2 ? 0 : third + 1) {
        const Place<T> here(a, t), there(a, t + step);         // `there` is but an address if that row is none
        T *g = GRAD ? (T *)a.grad + t * a.ldg : nullptr;
        const bool alike = GRAD && (((uintptr_t)g ^ (uintptr_t)here.x) & 15) == 0;
        uint4 *to = (uint4 *)((uintptr_t)g & ~(uintptr_t)15);
        uint32_t *taken = taken_twice + turn * words;
        const int n = now.n;
        const bool entry = tid < MANY && tid < n, more = n > MANY;             // more entries than are staged
        const int edges = (here.off > 0 ? 1 : 0) | ((here.off + a.ncols) % N ? here.all > 1 ? 2 : 1 : 0);      // granules that are not all the row's
        auto log_p = [&](float v, float ref) { return REST ? fmaf(v, a.c, -ref) : (v - ref) * a.c; };
        auto column = [&](int e) { return e < MANY ? staged.col[third][e] : a.crd[now.lo + e]; };
        auto value = [&](int e) { return e < MANY ? (float)staged.z[third][e] : (float)((const TV *)a.val)[now.lo + e]; };
        auto inside = [&](int64_t col) { return col >= 0 && col < a.ncols; };
        bool counts = false, first = false;        // first: of the granule's entries, this thread's is
        int mine = 0;                              // the granule that the thread takes by itself
        Seen own = {MINUS_INF, MINUS_INF, 0.0f, 0.0f, 0.0f, MINUS_INF, 0.0f, 0.0f};

        wait_copies_but(ring);                     // the entries are there: they were asked for before the chunks in the ring
        if (n > 0) {
            if (warp * 32 < n) {
                float x = MINUS_INF;
                bool in = false;
                if (entry) {
                    const int64_t col = staged.col[third][tid];
                    own.z = (float)staged.z[third][tid];
                    in = inside(col);
                    if (in) {
                        mine = here.granule_of(col);
                        const int prev = tid ? staged.prev[third][tid] : -1;
                        first = prev < 0 || here.granule_of(prev) != mine;
                        if (first) atomicOr(&taken[mine >> 5], 1u << (mine & 31));
                        x = to_float(((const T *)&staged.granule[turn][tid])[(here.off + (int)col) % N]);
                    }
                }
                own.x = x;
                if (more)
                    for (int e = MANY + tid; e < n; e += THREADS) {
                        const int64_t col = column(e);
                        own.z = max_nan(own.z, value(e));
                        if (inside(col)) {
                            own.x = max_nan(own.x, to_float(here.x[col]));
                            const int i = here.granule_of(col);
                            atomicOr(&taken[i >> 5], 1u << (i & 31));
                        }
                    }
                own.z = warp_max(own.z);
                own.x = warp_max(own.x);
                const float ref = REST ? now.lse * LOG2E : own.z, x0 = own.x == MINUS_INF ? 0.0f : own.x;
                auto take = [&](float ze, bool in, float xe) {
                    const float lp = log_p(ze, ref), p = exp2_fast(lp);
                    own.p += p;
                    if (!(p <= 0.0f)) own.plogp += p * lp;
                    if (!in) own.pu = __int_as_float(0x7fffffff);
                    else if (!(p <= 0.0f)) own.pu += p * ((xe - x0) * a.c);
                };
                if (own.z != MINUS_INF) {
                    if (entry) take((float)staged.z[third][tid], in, x);
                    if (more)
                        for (int e = MANY + tid; e < n; e += THREADS) {
                            const int64_t col = column(e);
                            take(value(e), inside(col), inside(col) ? to_float(here.x[col]) : 0.0f);
                        }
                }
                own.p = warp_sum(own.p);
                own.plogp = warp_sum(own.plogp);
                own.pu = warp_sum(own.pu);
            }
            if (edges) {                           // taken by the last two threads, unless an entry's thread does
                const int i = tid == THREADS - 1 ? 0 : here.all - 1;
                if ((tid == THREADS - 1 && edges & 1) || (tid == THREADS - 2 && edges & 2)) atomicOr(&taken[i >> 5], 1u << (i & 31));
            }
            if (lane == 0) seen[turn][warp] = own;
        }
        __syncthreads();
        if (n > 0)
            for (int i = 0; i < WARPS && i * 32 < n; i++) counts |= seen[turn][i].z != MINUS_INF;
        {
            uint32_t *before = taken_twice + (turn ^ 1) * words;               // the row before is done with it
            for (int i = tid; i < words; i += THREADS) before[i] = 0;
        }
        // what is to come
        copy_entry_granules(next, third == 2 ? 0 : third + 1, turn ^ 1, there);
        copy_entries(later, third == 0 ? 2 : third - 1);
        asm volatile("cp.async.commit_group;" ::: "memory");
        const Row after(a, t + 3 * step);
        const int64_t next_end = end_of(next);

        // the thread's edge, if no entry lies in it
        int edge = -1;
        if (counts && edges && tid >= THREADS - 2) {
            const int i = tid == THREADS - 1 ? 0 : here.all - 1;
            if (edges & (tid == THREADS - 1 ? 1 : 2) && !(inside(end) && here.granule_of(end) == i)) edge = i;
        }
        // f(granule's number, its 16 bytes, its first entry): each granule that the thread takes by itself
        auto alone = [&](auto f) {
            if (first) f(mine, staged.granule[turn][tid], tid);
            if (more)
                for (int e = MANY + tid; e < n; e += THREADS) {
                    const int64_t col = column(e), prev = column(e - 1);
                    if (!inside(col)) continue;
                    const int i = here.granule_of(col);
                    if (!inside(prev) || here.granule_of(prev) != i) f(i, here.from[i], e);
                }
            if (edge >= 0) f(edge, here.from[edge], n);
        };
        float loss = 0.0f;
        if (!counts) {
            left = 0;                              // what is in the ring of this row has no use, and the rest is not copied
            for (int c = 0; c < chunks + again; c++) {
                use = use + CHUNK == use_end ? use_begin : use + CHUNK;
                copy_next(here, false, there, next.n > 0);
            }
            if (GRAD)
                for (int i = tid; i < here.all; i += THREADS) {
                    const int col = i * N - here.off;
                    if (alike && col >= 0 && col + N <= a.ncols) {
                        to[i] = make_uint4(0, 0, 0, 0);
                    } else {
                        for (int k = 0; k < N; k++)
                            if (col + k >= 0 && col + k < a.ncols) g[col + k] = from_float<T>(0.0f);
                    }
                }
            __syncthreads();                       // the bitmap is clear
        } else {
            Sums sum(a.c);
            // of a chunk, which of the warp's 4 x 32 granules are others', or none: `rows` is what is left of the row from the warp's first
            auto left_out = [&](const uint4 *taken4, int rows) {
                uint4 w = *taken4;
                if (rows < BATCH * 32) {
                    auto none = [&](int k) { return rows >= 32 * (k + 1) ? 0u : rows <= 32 * k ? ~0u : ~0u << (rows - 32 * k); };
                    w.x |= none(0);
                    w.y |= none(1);
                    w.z |= none(2);
                    w.w |= none(3);
                }
                return w;
            };
            const uint4 *taken4 = (const uint4 *)taken + warp;
            int rows = here.all - warp * (BATCH * 32);
            for (int c = 0; c < chunks; c++) {
                // behind its own copy: the rest of the ring, or of the row if that stays, and the entries to come, if they were asked for after it
                wait_copies_but((GRAD ? min(ring, chunks - c) : ring) - 1 + (c < ring));
                const Granule<T> *from = use;
                use = use + CHUNK == use_end ? use_begin : use + CHUNK;
                if (rows > 0) {
                    Granule<T> v[BATCH];
#pragma unroll
                    for (int k = 0; k < BATCH; k++) v[k] = from[k * 32];
                    const uint4 out = left_out(taken4, rows);
                    if (out.x | out.y | out.z | out.w) {
                        const uint32_t w[BATCH] = {out.x, out.y, out.z, out.w};
#pragma unroll
                        for (int k = 0; k < BATCH; k++)
                            if (w[k] >> lane & 1) v[k] = Granule<T>::least();
                    }
                    sum.raise(to_float(largest(most_of(most_of(v[0].most(), v[1].most()), most_of(v[2].most(), v[3].most())))));
                    if (sum.u.near) {
#pragma unroll
                        for (int k = 0; k < BATCH; k++) sum.add_near(v[k]);
                    } else {
#pragma unroll 1
                        for (int k = 0; k < BATCH; k++)
                            if (lane + k * 32 < rows && !(((const uint32_t *)taken4)[k] >> lane & 1)) sum.add_any(from[k * 32]);
                    }
                }
                taken4 += CHUNK / (BATCH * 32);
                rows -= CHUNK;
                if (!GRAD || c < again) {
                    asm volatile("" ::"f"(sum.s.x), "f"(sum.s.y) : "memory");          // the slot has been read
                    copy_next(here, true, there, next.n > 0);
                }
            }
            alone([&](int i, uint4 bytes, int e) {
                Granule<T> v = here.masked(bytes, i, a.ncols);
                sum.raise(to_float(largest(v.most())));
                if (REST) {
                    T *elem = (T *)&v.w;
                    unsigned stored = 0;
                    for (; e < n; e++) {
                        const int64_t col = column(e);
                        if (!inside(col) || here.granule_of(col) != i) break;
                        stored |= 1u << ((here.off + (int)col) % N);
                    }
#pragma unroll
                    for (int k = 0; k < N; k++)
                        if (stored >> k & 1) {
                            sum.stored += exp2_fast(sum.u.of(to_float(elem[k])));
                            elem[k] = from_float<T>(MINUS_INF);
                        }
                }
                sum.add_any(v);
            });
            {
                const float m = warp_max(sum.m);
                const float f = sum.m == MINUS_INF ? 0.0f : exp2_fast(sum.u.to(Exponent(m, a.c)));
                const float others = warp_sum((sum.s.x + sum.s.y) * f), stored = REST ? warp_sum(sum.stored * f) : 0.0f;
                if (lane == 0) {
                    seen[turn][warp].m = m;
                    seen[turn][warp].others = others;
                    seen[turn][warp].stored = stored;
                }
            }
            __syncthreads();
            // the row's figures, in every warp: a lane per warp of the CTA
            const Seen of = lane < WARPS ? seen[turn][lane] : Seen{MINUS_INF, MINUS_INF, 0.0f, 0.0f, 0.0f, MINUS_INF, 0.0f, 0.0f};
            const Exponent top(warp_max(of.m), a.c);
            const float f = of.m == MINUS_INF ? 0.0f : exp2_fast(Exponent(of.m, a.c).to(top));
            const float others = warp_sum(of.others * f), stored = REST ? warp_sum(of.stored * f) : 0.0f, total = REST ? others + stored : others;
            float rescale = 1.0f, shift = 0.0f, zref = 0.0f;
            if (REST) {
                zref = now.lse * LOG2E;
            } else {
                zref = warp_max(of.z);
                shift = of.z == MINUS_INF ? 0.0f : (of.z - zref) * a.c;
                rescale = of.z == MINUS_INF ? 0.0f : exp2_fast(shift);
            }
            const float p = warp_sum(of.p * rescale), left = REST ? fmaxf(0.0f, 1.0f - p) : 0.0f, inv = REST ? 1.0f : 1.0f / p;
            if (warp == 0) {
                float x0 = warp_max(of.x);
                if (x0 == MINUS_INF) x0 = 0.0f;
                float plogp = 0.0f, pu = 0.0f;
                if (of.p * rescale != 0.0f) {
                    plogp = (of.plogp + of.p * shift) * rescale;
                    pu = (of.pu + of.p * (((of.x == MINUS_INF ? 0.0f : of.x) - x0) * a.c)) * rescale;
                } else if (of.pu != of.pu) {
                    pu = of.pu;                    // a column outside the matrix
                }
                plogp = warp_sum(plogp);
                pu = warp_sum(pu);
                // log2 of q: (x - x0) c + (x0 - top) c - log2(total)
                const float l2 = (total == 0.0f ? 0.0f : log2f(total)) - top.of(x0);
                loss = REST ? plogp - pu + p * l2 + (left > 0.0f ? left * (log2f(left) - log2f(others / total)) : 0.0f)
                            : (plogp - pu) * inv - log2f(p) + l2;
            }
            if (GRAD) {
                const float by = now.w * a.by, part_of = total == 0.0f ? 0.0f : by / total;        // total 0: every logit is -inf
                const float factor = left > 0.0f && others > 0.0f ? part_of * (1.0f - left * (total / others)) : part_of;
                alone([&](int i, uint4 bytes, int e) {
                    const Granule<T> x = here.masked(bytes, i, a.ncols);
                    float v[N], minus[N];
                    x.unpack(v);
                    unsigned stored = 0;
#pragma unroll
                    for (int k = 0; k < N; k++) minus[k] = 0.0f;
                    for (; e < n; e++) {           // repeated columns add up
                        const int64_t col = column(e);
                        if (!inside(col) || here.granule_of(col) != i) break;
                        const int at = (here.off + (int)col) % N;
                        const float pe = exp2_fast(log_p(value(e), zref));
                        stored |= 1u << at;
#pragma unroll
                        for (int k = 0; k < N; k++)
                            if (k == at) minus[k] += pe;
                    }
#pragma unroll
                    for (int k = 0; k < N; k++) {
                        const int col = i * N + k - here.off;
                        const float qk = exp2_fast(top.of(v[k]));
                        if (col >= 0 && col < a.ncols) g[col] = from_float<T>(stored >> k & 1 ? part_of * qk - by * (minus[k] * inv) : factor * qk);
                    }
                });
                // the chunks in the ring, then the ones before them, copied again
                const float2 factor2 = make_float2(factor, factor);
                taken4 = (const uint4 *)taken + again * (CHUNK / (BATCH * 32)) + warp;
                rows = here.all - warp * (BATCH * 32) - again * CHUNK;
                uint4 *out16 = to + again * CHUNK + mine0;
                for (int c = 0; c < chunks; c++) {
                    if (c >= ring) {
                        wait_copies_but(ring - 1);
                        if (c == ring) {
                            taken4 = (const uint4 *)taken + warp;
                            rows = here.all - warp * (BATCH * 32);
                            out16 = to + mine0;
                        }
                    }
                    const Granule<T> *from = use;
                    use = use + CHUNK == use_end ? use_begin : use + CHUNK;
                    if (rows > 0) {
                        if (alike && top.near) {
                            Granule<T> x[BATCH];
#pragma unroll
                            for (int k = 0; k < BATCH; k++) x[k] = from[k * 32];
                            const uint4 out = left_out(taken4, rows);
                            const uint32_t w[BATCH] = {out.x, out.y, out.z, out.w};
#pragma unroll
                            for (int k = 0; k < BATCH; k++) {
                                float2 v[N / 2];
                                x[k].unpack(v);
#pragma unroll
                                for (int j = 0; j < N / 2; j++) {
                                    v[j] = top.of(v[j]);
                                    v[j] = mul2(make_float2(exp2_fast(v[j].x), exp2_fast(v[j].y)), factor2);
                                }
                                x[k].pack(v);
                                if (!(w[k] >> lane & 1)) out16[k * 32] = x[k].w;
                            }
                        } else {
#pragma unroll 1
                            for (int k = 0; k < BATCH; k++) {
                                if (lane + k * 32 >= rows || ((const uint32_t *)taken4)[k] >> lane & 1) continue;
                                float v[N];
                                from[k * 32].unpack(v);
                                T *each = g + (int)(out16 + k * 32 - to) * N - here.off;
#pragma unroll
                                for (int j = 0; j < N; j++) each[j] = from_float<T>(factor * exp2_fast(top.of(v[j])));
                            }
                        }
                    }
                    taken4 += CHUNK / (BATCH * 32);
                    rows -= CHUNK;
                    out16 += CHUNK;
                    copy_next(here, true, there, next.n > 0);  // the slot has been read
                }
            }
        }
        if (tid == 0) a.rows[t] = loss * LN2;
        now = next;
        next = later;
        later = after;
        end = next_end;
    }
    wait_copies();
}

template <typename T, typename TV, int THREADS, bool REST, bool GRAD>
static int launch_rows(const DistillArgs &a, int chunks, cudaStream_t st)
{
    constexpr size_t on_sm = 228 * 1024, of_system = 1024, chunk = (size_t)BATCH * THREADS * 16;
    constexpr size_t most = on_sm / (512 / THREADS) - of_system - sizeof(Staged<TV, THREADS / 2>) - 2 * (THREADS / 32) * sizeof(Seen) - 64;
    const size_t bits = (size_t)chunks * BATCH * THREADS / 32 * 8;
    int ring = chunks < SLOTS ? chunks : SLOTS;
    while (ring > 1 && ring * chunk + bits > most) ring--;
    if (ring * chunk + bits > most) return fail("distill_loss: rows of %d columns are too long", a.ncols);
    const size_t smem = ring * chunk + bits;
    auto kernel = distill_rows_kernel<T, TV, THREADS, REST, GRAD>;
    CB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    const int64_t ctas = (int64_t)sm_count() * (512 / THREADS);
    kernel<<<(unsigned)(a.nrows < ctas ? a.nrows : ctas), THREADS, smem, st>>>(a, chunks, ring);
    CB_LAUNCH_CHECK();
    CB_CUDA(launch_behind(distill_sum_kernel, dim3(1), 1024, 0, st, a));
    return 0;
}

template <typename T, typename TV, int THREADS>
static int launch_rows(const DistillArgs &a, int chunks, cudaStream_t st)
{
    if (a.lse) return a.grad ? launch_rows<T, TV, THREADS, true, true>(a, chunks, st) : launch_rows<T, TV, THREADS, true, false>(a, chunks, st);
    return a.grad ? launch_rows<T, TV, THREADS, false, true>(a, chunks, st) : launch_rows<T, TV, THREADS, false, false>(a, chunks, st);
}

// The smallest CTAs that hold a row: 512 threads on an SM all the same, and the more rows at a time the less their barriers cost.
template <typename T, typename TV>
static int launch_rows(const DistillArgs &a, cudaStream_t st)
{
    constexpr int N = Granule<T>::N;
    const bool alike = a.ldx * (int64_t)sizeof(T) % 16 == 0;   // granules of a row, where it starts
    const int64_t all = (a.ncols + (alike ? (int)((uintptr_t)a.x % 16 / sizeof(T)) : N - 1) + N - 1) / N;
    if (all <= 128 * BATCH * SLOTS) return launch_rows<T, TV, 128>(a, (int)ceil_div(all, 128 * BATCH), st);
    if (all <= 256 * BATCH * SLOTS) return launch_rows<T, TV, 256>(a, (int)ceil_div(all, 256 * BATCH), st);
    return launch_rows<T, TV, 512>(a, (int)ceil_div(all, 512 * BATCH), st);
}

template <typename T>
int distill_by_rows(DistillArgs a, int val_bytes, cudaStream_t st)
{
    return val_bytes == 4 ? launch_rows<T, float>(a, st) : launch_rows<T, double>(a, st);
}
template int distill_by_rows<__nv_bfloat16>(DistillArgs, int, cudaStream_t);
template int distill_by_rows<__half>(DistillArgs, int, cudaStream_t);
template int distill_by_rows<float>(DistillArgs, int, cudaStream_t);

}  // namespace cb200
