// kv_page_ops_sm100.cu — pages that change hands without a step: sequences that begin as copies of others, that are cut back or end, pools that are made dense, and
// the bytes that follow (kv_page_fork, kv_page_release, kv_page_compact, kv_page_copy, include/fp8_block.h).
//
// The first three are a few dependent passes over lengths, tables and pages with next to nothing to compute, so what they cost is the waits between the passes.  One
// cluster of eight CTAs makes all of them: its barrier takes less than a microsecond, where a launch behind another takes two.  Counts meet in distributed shared memory.
// Ranks come from counts in the order of pages or sequences, never from who is first, so results do not depend on timing.
// Measured in CUDA graphs, us: fork of a few tens of sequences 6.2, of hundreds 7.8; release 6.4 for 32 sequences, 13.2 for 2048 with windows; compact 8.8 for a small pool, 15.4 for 23000 pages.
#include <cuda_runtime.h>
#include <stdint.h>

#include <initializer_list>

#include "../../include/fp8_block.h"
#include "pdl.cuh"
#include "row_items.cuh"

namespace {

using namespace sm100;

constexpr int CTAS = 8;   // the portable size of a cluster
constexpr int THREADS = 1024, WARPS = THREADS / 32, ALL_WARPS = CTAS * WARPS, ALL_THREADS = CTAS * THREADS;

__device__ __forceinline__ int cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return (int)r;
}
// What any thread of the cluster has written before, every thread sees behind it.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Exclusive sum over the cluster's warps in order of one number a warp (the same in its lanes), and the total.  A cluster_sync in passing, and one has to lie ahead of
// it: every CTA must run before its shared memory is written.  Each `sh` serves once.
struct Before {
    int warp, total;
};
__device__ __forceinline__ Before cluster_sum(int x, int (*sh)[WARPS + CTAS]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = cluster_rank();
    if (lane == 0) (*sh)[warp] = x;
    __syncthreads();
    if (warp == 0) {
        const int mine = __reduce_add_sync(0xffffffffu, (*sh)[lane]);
        if (lane < CTAS) {
            const uint32_t at = (uint32_t)__cvta_generic_to_shared(&(*sh)[WARPS + rank]);
            asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, %1;\n\tst.shared::cluster.u32 [a], %2;\n\t}" ::"r"(at), "r"(lane), "r"(mine) : "memory");
        }
    }
    __syncwarp();
    cluster_sync();
    const int of_warp = lane < warp ? (*sh)[lane] : 0, of_cta = lane < CTAS ? (*sh)[WARPS + lane] : 0;
    Before b;
    b.warp = __reduce_add_sync(0xffffffffu, of_warp + (lane < rank ? of_cta : 0));
    b.total = __reduce_add_sync(0xffffffffu, of_cta);
    return b;
}
__device__ __forceinline__ int lanes_below(uint32_t votes) { return __popc(votes & ((1u << (threadIdx.x & 31)) - 1u)); }

// what all three have in common.  Sequences and pages may be 2^31 - 1: a count that a step or a sum may carry past them has no sign.
struct Pages {
    const int32_t* lens;
    const int32_t* table;
    int batch, max_pages, num_pages, capacity;
    FastDiv page;
    __device__ __forceinline__ int length(int b) const { return min(max(ld_s32(lens + b), 0), capacity); }
    __device__ __forceinline__ int pages_of(int n) const { return n > 0 ? (int)page.div((uint32_t)n - 1u) + 1 : 0; }
    // pages that hold no key which a token behind n keys sees through a window (it sees those from n + 1 - window on)
    __device__ __forceinline__ int passed(int n, int window) const { return n >= window ? (int)page.div((uint32_t)(n - window) + 1u) : 0; }
    __device__ __forceinline__ bool inside(int p) const { return (uint32_t)p < (uint32_t)num_pages; }
    // entry i of a ring from place `from` on; from and i are below num_pages
    __device__ __forceinline__ int ring_at(int from, int i) const {
        const uint32_t at = (uint32_t)from + (uint32_t)i;
        return (int)(at < (uint32_t)num_pages ? at : at - (uint32_t)num_pages);
    }
    // Entries of the table's rows, side by side whatever their sequences: of sequence b the `count` ones that of(b) gives and at(j) places.  A warp has 32 sequences, one to a lane,
    // and takes their entries 32 at a time; where sequences are few, several warps take turns at the same 32.
    // of(b): what is known of a sequence, with int count; use(b, s, i): entry i of sequence b, of which s = of(b)
    template <class Of, class Use>
    __device__ __forceinline__ void each_entry(Of&& of, Use&& use) const {
        const int lane = threadIdx.x & 31, warp = cluster_rank() * WARPS + (threadIdx.x >> 5), sets = (int)(((uint32_t)batch + 31u) / 32u), share = max(ALL_WARPS / max(sets, 1), 1);
        for (int item = warp; item < sets * share; item += ALL_WARPS) {
            const int set = item / share;
            const bool is_one = 32u * (uint32_t)set + (uint32_t)lane < (uint32_t)batch;
            auto mine = of(is_one ? 32 * set + lane : batch - 1);
            const int count = is_one ? mine.count : 0;
            long long upto = count;   // entries of the lanes up to this one
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            const long long total = __shfl_sync(0xffffffffu, upto, 31);
            for (long long e0 = 32 * (item - set * share); e0 < total; e0 += 32 * share) {
                const long long e = e0 + lane;
                int owner = 0;   // the lanes whose entries end at or before e
#pragma unroll
                for (int step = 16; step; step >>= 1)
                    if (__shfl_sync(0xffffffffu, upto, owner + step - 1) <= e) owner += step;
                owner = min(owner, 31);
                auto s = mine.from_lane(owner);
                const long long before = __shfl_sync(0xffffffffu, upto - count, owner);
                if (e < total) use(32 * set + owner, s, (int)(e - before));
            }
        }
    }
    // use(p, value): all pages, those of a warp one behind another, by all its lanes (value: load(p), or `none` past the end); four loads of a lane on their way
    template <class Load, class Use>
    __device__ __forceinline__ void each_page(int none, Load&& load, Use&& use) const {
        const long long per = ((long long)num_pages + ALL_THREADS - 1) / ALL_THREADS * 32;   // of a warp
        const long long first = (long long)(cluster_rank() * WARPS + (threadIdx.x >> 5)) * per;
        const int end = (int)min(first + per, (long long)num_pages);
        for (long long p0 = first; p0 < end; p0 += 128) {
            int value[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const long long p = p0 + 32 * k + (threadIdx.x & 31);
                value[k] = p < end ? load((int)p) : none;
            }
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (p0 + 32 * k < end) use((int)((uint32_t)(p0 + 32 * k) + (threadIdx.x & 31)), value[k]);   // (past the end, where the value is `none`, perhaps below zero)
        }
    }
};
struct Ring {
    int head, count;
    __device__ __forceinline__ Ring(const int32_t* state, int num_pages) {
        head = (int)((uint32_t)max(ld_s32(state), 0) % (uint32_t)num_pages);
        count = min(max(ld_s32(state + 1), 0), num_pages);
    }
};
__device__ __forceinline__ void copy_shares(const Pages& a, const int32_t* from, int32_t* to) {
    if (from != to)
        for (uint32_t p = cluster_rank() * THREADS + threadIdx.x; p < (uint32_t)a.num_pages; p += ALL_THREADS) to[p] = ld_s32(from + p);
}
__device__ __forceinline__ int gone_of(const int32_t* gone, int b) { return gone ? max(ld_s32(gone + b), 0) : 0; }

// ------------------------------------------------------------------------------------------------------------------- fork
struct Fork : Pages {
    const int32_t *parent, *keep, *ring, *state, *shares, *gone;
    int32_t *table_out, *lens_out, *state_out, *shares_out, *gone_out, *taken, *copy_from, *copy_to, *copies;
    int window, sink_pages;
    // whether a copy of n keys (`full` whole pages and, part != 0, one more) lacks a page that it needs, where those behind the sinks start at `gone`: one that a token behind
    // it sees through the window or, of no window, the one that is to be copied
    __device__ __forceinline__ bool lacks(int n, int full, int part, int gone) const {
        if (window) return max(passed(n, window), sink_pages) < min(gone, full + (part != 0));
        return part && full >= sink_pages && full < gone;
    }
};

__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__(THREADS, 1) kv_page_fork_kernel(const Fork a) {
    __shared__ int sh[1][WARPS + CTAS];
    const int rank = cluster_rank(), lane = threadIdx.x & 31;
    cluster_sync();
    pdl_wait();
    pdl_trigger();
    const Ring ring(a.state, a.num_pages);
    copy_shares(a, a.shares, a.shares_out);
    // ---- what a fork wants: nothing is written over that another sequence's thread still reads
    const int run = (int)(((uint32_t)a.batch + (ALL_THREADS - 1u)) / ALL_THREADS);
    const long long first = (long long)(rank * THREADS + threadIdx.x) * run;
    const int b_begin = (int)min(first, (long long)a.batch), b_end = (int)min(first + run, (long long)a.batch);
    int needs = 0;
    for (int b = b_begin; b < b_end; b++) {
        const int p = ld_s32(a.parent + b);
        int n = -1;   // no fork
        if ((uint32_t)p < (uint32_t)a.batch && p != b && a.length(b) == 0) {
            n = a.length(p);
            if (a.keep) n = min(n, max(ld_s32(a.keep + b), 0));
            uint32_t full, part;
            a.page.divmod((uint32_t)n, full, part);
            if (a.lacks(n, (int)full, (int)part, gone_of(a.gone, p))) n = -1;
            else needs += part != 0;
        }
        a.taken[b] = n;
    }
    int before = needs;   // those of the lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += y;
    }
    const Before all = cluster_sum(__shfl_sync(0xffffffffu, before, 31), sh);
    before += all.warp - needs;
    // ---- the pages that are new
    for (int b = b_begin; b < b_end; b++) {
        const int n = a.taken[b], p = ld_s32(a.parent + b);
        uint32_t full = 0, part = 0;
        if (n >= 0) a.page.divmod((uint32_t)n, full, part);
        const int at = before;
        before += part != 0;
        const bool served = n >= 0 && (!part || at < ring.count);
        a.taken[b] = served ? n : 0;
        if (served) {
            a.lens_out[b] = n;
        } else if (a.lens_out != a.lens) {
            a.lens_out[b] = ld_s32(a.lens + b);
        }
        if (a.gone_out) {
            if (served) a.gone_out[b] = min(gone_of(a.gone, p), (int)full);
            else if (a.gone_out != a.gone) a.gone_out[b] = ld_s32(a.gone + b);
        }
        if (served && part) {
            const int fresh = ld_s32(a.ring + a.ring_at(ring.head, at));
            a.copy_from[at] = ld_s32(a.table + (size_t)p * a.max_pages + full);
            a.copy_to[at] = fresh;
            a.table_out[(size_t)b * a.max_pages + full] = fresh;
        }
    }
    if (rank == 0 && threadIdx.x == 0) {
        const int used = min(all.total, ring.count);
        a.state_out[0] = a.ring_at(ring.head, used == a.num_pages ? 0 : used);
        a.state_out[1] = ring.count - used;
        *a.copies = used;
    }
    cluster_sync();
    // ---- the pages that are shared: those in front of the sinks' end, then those from the first that has not gone
    struct Shared {
        int count, parent, sinks, skip;
        __device__ __forceinline__ Shared from_lane(int l) const {
            Shared s;
            s.count = 0;
            s.parent = __shfl_sync(0xffffffffu, parent, l);
            s.sinks = __shfl_sync(0xffffffffu, sinks, l);
            s.skip = __shfl_sync(0xffffffffu, skip, l);
            return s;
        }
    };
    a.each_entry(
        [&](int b) {
            Shared s;
            const int full = (int)a.page.div((uint32_t)ld_s32(a.taken + b));
            s.parent = full ? ld_s32(a.parent + b) : 0;
            const int gone = full ? gone_of(a.gone, s.parent) : 0;
            s.sinks = min(a.sink_pages, full);
            s.skip = max(min(gone, full) - s.sinks, 0);
            s.count = full - s.skip;
            return s;
        },
        [&](int b, const Shared& s, int i) {
            const int j = i < s.sinks ? i : i + s.skip, page = ld_s32(a.table + (size_t)s.parent * a.max_pages + j);
            a.table_out[(size_t)b * a.max_pages + j] = page;
            if (a.inside(page)) atomicAdd(a.shares_out + page, 1);
        });
}

// ---------------------------------------------------------------------------------------------------------------- release
struct Release : Pages {
    const int32_t *keep, *state, *shares, *gone;
    int32_t *ring, *lens_out, *state_out, *shares_out, *gone_out;
    int window, sink_pages;
};
struct Cut {
    int after, left;              // length and first page behind the sinks, then
    int held, gone, held_after;   // pages, and what has gone, before; pages then
    int count, n1, n2, from;      // pages given back: n1 from held_after on, n2 from `from`, the others from max(from, held_after) on
    __device__ __forceinline__ Cut() {}
    __device__ __forceinline__ Cut(const Release& a, int b) {
        const int n = a.length(b);
        after = a.keep ? min(n, max(ld_s32(a.keep + b), 0)) : n;
        held = a.pages_of(n);
        gone = gone_of(a.gone, b);
        held_after = a.pages_of(after);
        left = min(max(gone, a.window ? a.passed(after, a.window) : 0), held_after);
        // had: [0, sink_pages) and [gone, held); has: [0, sink_pages) and [left, held_after)
        n1 = max(min(a.sink_pages, held) - held_after, 0);
        from = max(gone, a.sink_pages);
        n2 = max(left - from, 0);
        count = n1 + n2 + max(held - max(from, held_after), 0);
    }
    __device__ __forceinline__ int page(int i) const { return i < n1 ? held_after + i : i < n1 + n2 ? from + i - n1 : max(from, held_after) + i - n1 - n2; }
    __device__ __forceinline__ Cut from_lane(int l) const {
        Cut c;
        c.held_after = __shfl_sync(0xffffffffu, held_after, l);
        c.n1 = __shfl_sync(0xffffffffu, n1, l);
        c.n2 = __shfl_sync(0xffffffffu, n2, l);
        c.from = __shfl_sync(0xffffffffu, from, l);
        return c;
    }
};

// A page that nobody has any more has less than zero sharers.
__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__(THREADS, 1) kv_page_release_kernel(const Release a) {
    __shared__ int sh[1][WARPS + CTAS];
    const int rank = cluster_rank();
    pdl_wait();
    pdl_trigger();
    const Ring ring(a.state, a.num_pages);
    if (a.shares != a.shares_out) {
        copy_shares(a, a.shares, a.shares_out);
        cluster_sync();
    }
    a.each_entry([&](int b) { return Cut(a, b); },
                 [&](int b, const Cut& c, int i) {
                     const int page = ld_s32(a.table + (size_t)b * a.max_pages + c.page(i));
                     if (a.inside(page)) atomicSub(a.shares_out + page, 1);
                 });
    cluster_sync();
    auto sharers = [&](int p) { return __ldcg(a.shares_out + p); };
    int mine = 0;
    a.each_page(0, sharers, [&](int, int n) { mine += __popc(__ballot_sync(0xffffffffu, n < 0)); });
    const Before all = cluster_sum(mine, sh);
    uint32_t at = (uint32_t)ring.count + (uint32_t)all.warp;
    a.each_page(0, sharers, [&](int p, int n) {
        const uint32_t votes = __ballot_sync(0xffffffffu, n < 0);
        if (n < 0) {
            const uint32_t i = at + lanes_below(votes);
            if (i < (uint32_t)a.num_pages) a.ring[a.ring_at(ring.head, (int)i)] = p;   // a ring holds all pages
            a.shares_out[p] = 0;
        }
        at += __popc(votes);
    });
    for (uint32_t b = rank * THREADS + threadIdx.x; b < (uint32_t)a.batch; b += ALL_THREADS) {
        const Cut c(a, (int)b);
        a.lens_out[b] = c.after;
        if (a.gone_out) a.gone_out[b] = c.left;
    }
    if (rank == 0 && threadIdx.x == 0) {
        a.state_out[0] = ring.head;
        a.state_out[1] = (int)min((uint32_t)ring.count + (uint32_t)all.total, (uint32_t)a.num_pages);
    }
}

// ---------------------------------------------------------------------------------------------------------------- compact
struct Compact : Pages {
    const int32_t *ring, *state, *shares;
    int32_t *table_out, *ring_out, *state_out, *shares_out, *moved_to, *copy_from, *copy_to, *copies;
};

__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__(THREADS, 1) kv_page_compact_kernel(const Compact a) {
    __shared__ int sh[2][WARPS + CTAS];
    const int thread = cluster_rank() * THREADS + threadIdx.x;
    pdl_wait();
    pdl_trigger();
    const Ring ring(a.state, a.num_pages);
    for (uint32_t p = thread; p < (uint32_t)a.num_pages; p += ALL_THREADS) a.moved_to[p] = 0;
    cluster_sync();
    for (uint32_t i = thread; i < (uint32_t)ring.count; i += ALL_THREADS) {
        const int p = ld_s32(a.ring + a.ring_at(ring.head, (int)i));
        if (a.inside(p)) a.moved_to[p] = -1;   // free
    }
    cluster_sync();
    // ---- the used pages are to be those below `used`: the others of them move to the free ones there, in order
    auto mark = [&](int p) { return __ldcg(a.moved_to + p); };   // 0: used
    int mine = 0;
    a.each_page(-1, mark, [&](int, int m) { mine += __popc(__ballot_sync(0xffffffffu, m == 0)); });
    const Before of_used = cluster_sum(mine, &sh[0]);
    const int used = of_used.total;
    mine = 0;
    a.each_page(-1, mark, [&](int p, int m) { mine += __popc(__ballot_sync(0xffffffffu, m == 0 && p >= used)); });
    const Before of_movers = cluster_sum(mine, &sh[1]);
    int movers = of_movers.warp, below = of_used.warp;
    a.each_page(1, mark, [&](int p, int m) {
        const bool moves = m == 0 && p >= used;
        const uint32_t votes = __ballot_sync(0xffffffffu, m == 0), moving = __ballot_sync(0xffffffffu, moves);
        if (moves) a.copy_from[movers + lanes_below(moving)] = p;
        if (m < 0 && p < used) a.copy_to[p - (below + lanes_below(votes))] = p;
        below += __popc(votes);
        movers += __popc(moving);
    });
    cluster_sync();
    movers = of_movers.warp;
    a.each_page(1, mark, [&](int p, int m) {
        const bool moves = m == 0 && p >= used;
        const uint32_t moving = __ballot_sync(0xffffffffu, moves);
        if (m == 0) {
            const int to = moves ? __ldcg(a.copy_to + movers + lanes_below(moving)) : p;
            a.moved_to[p] = to;
            a.shares_out[to] = ld_s32(a.shares + p);
        }
        if (m <= 0 && p >= used) a.shares_out[p] = 0;
        movers += __popc(moving);
    });
    cluster_sync();
    struct Held {
        int count;
        __device__ __forceinline__ Held from_lane(int) const { return *this; }
    };
    a.each_entry([&](int b) { return Held{a.pages_of(a.length(b))}; },
                 [&](int b, const Held&, int j) {
                     const size_t at = (size_t)b * a.max_pages + j;
                     const int p = ld_s32(a.table + at);
                     a.table_out[at] = a.inside(p) ? __ldcg(a.moved_to + p) : -1;
                 });
    for (uint32_t i = thread; i < (uint32_t)a.num_pages; i += ALL_THREADS) a.ring_out[i] = i < (uint32_t)(a.num_pages - used) ? used + (int)i : -1;
    if (thread == 0) {
        a.state_out[0] = 0;
        a.state_out[1] = a.num_pages - used;
        *a.copies = of_movers.total;
    }
}

// ------------------------------------------------------------------------------------------------------------------- copy
constexpr int COPY_THREADS = 256, COPY_WIDE = 4, COPY_BYTES = COPY_THREADS * COPY_WIDE * 16;   // bytes that a CTA has in flight
constexpr int COPY_POOLS = 64;   // of a launch
struct Copy {
    const int32_t *from, *to, *copies;
    int most, num_pages, pools;
    int pieces;   // of one page, in all pools
    uint8_t* pool[COPY_POOLS];
    long long page_bytes[COPY_POOLS];
    int first_piece[COPY_POOLS];
};
// Bound by memory: 751 MB read and written in 129 us (5.8 TB/s); 76 MB, which L2 holds in part, in 8.4.
__global__ void __launch_bounds__(COPY_THREADS) kv_page_copy_kernel(const __grid_constant__ Copy a) {
    pdl_wait();
    pdl_trigger();
    const long long items = (long long)min(max(ld_s32(a.copies), 0), a.most) * a.pieces;
    for (long long item = blockIdx.x; item < items; item += gridDim.x) {
        const int i = (int)(item / a.pieces), piece = (int)(item - (long long)i * a.pieces);
        const int from = ld_s32(a.from + i), to = ld_s32(a.to + i);
        if ((uint32_t)from >= (uint32_t)a.num_pages || (uint32_t)to >= (uint32_t)a.num_pages || from == to) continue;
        int k = 0;
        for (int step = COPY_POOLS / 2; step; step >>= 1)
            if (k + step < a.pools && a.first_piece[k + step] <= piece) k += step;
        const long long bytes = a.page_bytes[k], at = (long long)(piece - a.first_piece[k]) * COPY_BYTES + threadIdx.x * 16;
        const uint8_t* src = a.pool[k] + from * bytes;
        uint8_t* dst = a.pool[k] + to * bytes;
        uint4 x[COPY_WIDE];
#pragma unroll
        for (int w = 0; w < COPY_WIDE; w++)
            if (at + w * (COPY_THREADS * 16) < bytes) x[w] = ld128(src + at + w * (COPY_THREADS * 16));
#pragma unroll
        for (int w = 0; w < COPY_WIDE; w++)
            if (at + w * (COPY_THREADS * 16) < bytes) *reinterpret_cast<uint4*>(dst + at + w * (COPY_THREADS * 16)) = x[w];
    }
}

// ------------------------------------------------------------------------------------------------------------------- host
bool words(std::initializer_list<const void*> pointers) {
    for (const void* p : pointers)
        if (reinterpret_cast<uintptr_t>(p) & 3) return false;
    return true;
}
bool fill(Pages& a, const int32_t* lens, const int32_t* table, int batch, int max_pages, int page_size, int num_pages) {
    if (batch < 0 || max_pages <= 0 || page_size <= 0 || num_pages <= 0) return false;
    if ((long long)page_size * max_pages > 0x7fffffffLL || (long long)page_size * num_pages > 0x7fffffffLL) return false;
    a.lens = lens;
    a.table = table;
    a.batch = batch;
    a.max_pages = max_pages;
    a.num_pages = num_pages;
    a.capacity = page_size * max_pages;
    a.page = FastDiv((uint32_t)page_size);
    return true;
}
int pages_behind(int tokens, int page_size) { return (int)(((long long)tokens + page_size - 1) / page_size); }

}  // namespace

extern "C" int kv_page_fork(const kv_page_fork_args_t* g) {
    if (!g || !g->lens || !g->parent || !g->block_table || !g->ring || !g->ring_state || !g->shares || !g->lens_out || !g->ring_state_out || !g->shares_out || !g->taken ||
        !g->copy_from || !g->copy_to || !g->copies || !g->gone != !g->gone_out || g->window < 0 || g->sinks < 0)
        return (int)cudaErrorInvalidValue;
    if (!words({g->lens, g->parent, g->keep, g->block_table, g->ring, g->ring_state, g->shares, g->gone, g->lens_out, g->ring_state_out, g->shares_out, g->gone_out, g->taken,
                g->copy_from, g->copy_to, g->copies}))
        return (int)cudaErrorInvalidValue;
    Fork a;
    if (!fill(a, g->lens, g->block_table, g->batch, g->max_pages_per_seq, g->page_size, g->num_pages)) return (int)cudaErrorInvalidValue;
    a.parent = g->parent; a.keep = g->keep; a.ring = g->ring; a.state = g->ring_state; a.shares = g->shares; a.gone = g->gone;
    a.table_out = g->block_table; a.lens_out = g->lens_out; a.state_out = g->ring_state_out; a.shares_out = g->shares_out; a.gone_out = g->gone_out; a.taken = g->taken;
    a.copy_from = g->copy_from; a.copy_to = g->copy_to; a.copies = g->copies;
    a.window = g->window;
    a.sink_pages = pages_behind(g->sinks, g->page_size);
    return (int)launch_pdl(kv_page_fork_kernel, dim3(CTAS), dim3(THREADS), 0, (cudaStream_t)g->stream, a);
}

extern "C" int kv_page_release(const kv_page_release_args_t* g) {
    if (!g || !g->lens || !g->block_table || !g->ring || !g->ring_state || !g->shares || !g->lens_out || !g->ring_state_out || !g->shares_out || !g->gone != !g->gone_out ||
        g->window < 0 || g->sinks < 0 || (g->window > 0 && !g->gone))
        return (int)cudaErrorInvalidValue;
    if (!words({g->lens, g->keep, g->block_table, g->ring, g->ring_state, g->shares, g->gone, g->lens_out, g->ring_state_out, g->shares_out, g->gone_out}))
        return (int)cudaErrorInvalidValue;
    Release a;
    if (!fill(a, g->lens, g->block_table, g->batch, g->max_pages_per_seq, g->page_size, g->num_pages)) return (int)cudaErrorInvalidValue;
    a.keep = g->keep; a.ring = g->ring; a.state = g->ring_state; a.shares = g->shares; a.gone = g->gone;
    a.lens_out = g->lens_out; a.state_out = g->ring_state_out; a.shares_out = g->shares_out; a.gone_out = g->gone_out;
    a.window = g->window;
    a.sink_pages = pages_behind(g->sinks, g->page_size);
    return (int)launch_pdl(kv_page_release_kernel, dim3(CTAS), dim3(THREADS), 0, (cudaStream_t)g->stream, a);
}

extern "C" int kv_page_compact(const kv_page_compact_args_t* g) {
    if (!g || !g->lens || !g->block_table || !g->ring || !g->ring_state || !g->shares || !g->block_table_out || !g->ring_out || !g->ring_state_out || !g->shares_out ||
        !g->moved_to || !g->copy_from || !g->copy_to || !g->copies)
        return (int)cudaErrorInvalidValue;
    if (!words({g->lens, g->block_table, g->ring, g->ring_state, g->shares, g->block_table_out, g->ring_out, g->ring_state_out, g->shares_out, g->moved_to, g->copy_from, g->copy_to,
                g->copies}))
        return (int)cudaErrorInvalidValue;
    Compact a;
    if (!fill(a, g->lens, g->block_table, g->batch, g->max_pages_per_seq, g->page_size, g->num_pages)) return (int)cudaErrorInvalidValue;
    a.ring = g->ring; a.state = g->ring_state; a.shares = g->shares;
    a.table_out = g->block_table_out; a.ring_out = g->ring_out; a.state_out = g->ring_state_out; a.shares_out = g->shares_out;
    a.moved_to = g->moved_to; a.copy_from = g->copy_from; a.copy_to = g->copy_to; a.copies = g->copies;
    return (int)launch_pdl(kv_page_compact_kernel, dim3(CTAS), dim3(THREADS), 0, (cudaStream_t)g->stream, a);
}

extern "C" int kv_page_copy(const kv_page_copy_args_t* g) {
    if (!g || !g->copy_from || !g->copy_to || !g->copies || g->most < 0 || g->num_pages <= 0 || g->num_pools < 0 || (g->num_pools > 0 && !g->pools)) return (int)cudaErrorInvalidValue;
    if (!words({g->copy_from, g->copy_to, g->copies})) return (int)cudaErrorInvalidValue;
    for (int k = 0; k < g->num_pools; k++) {
        const kv_page_pool_t& p = g->pools[k];
        if (!p.data || p.page_bytes <= 0 || ((reinterpret_cast<uintptr_t>(p.data) | (uintptr_t)p.page_bytes) & 15) || p.page_bytes > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    }
    if (g->most == 0) return (int)cudaSuccess;
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    for (int k0 = 0; k0 < g->num_pools; k0 += COPY_POOLS) {
        Copy a = {};
        a.from = g->copy_from; a.to = g->copy_to; a.copies = g->copies;
        a.most = g->most;
        a.num_pages = g->num_pages;
        a.pools = g->num_pools - k0 < COPY_POOLS ? g->num_pools - k0 : COPY_POOLS;
        long long pieces = 0;
        for (int k = 0; k < a.pools; k++) {
            a.pool[k] = static_cast<uint8_t*>(g->pools[k0 + k].data);
            a.page_bytes[k] = g->pools[k0 + k].page_bytes;
            a.first_piece[k] = (int)pieces;
            pieces += (a.page_bytes[k] + COPY_BYTES - 1) / COPY_BYTES;
        }
        a.pieces = (int)pieces;   // at most 64 * 2^17
        const long long items = pieces * g->most, most_ctas = 8LL * sms;
        const cudaError_t e = launch_pdl(kv_page_copy_kernel, dim3((unsigned)(items < most_ctas ? items : most_ctas)), dim3(COPY_THREADS), 0, (cudaStream_t)g->stream, a);
        if (e != cudaSuccess) return (int)e;
    }
    return (int)cudaSuccess;
}
