// kv_page_ops_sm100.cu — pages that change hands without a step: sequences that begin as copies of others, that are cut back or end, pools that are made dense, and
// the bytes that follow (kv_page_fork, kv_page_release, kv_page_compact, kv_page_copy, include/fp8_block.h).
//
// The first three are a few dependent passes over lengths, tables and pages with next to nothing to compute, so what they cost is the waits between the passes.  One
// cluster of eight CTAs makes all of them: its barrier takes less than a microsecond, where a launch behind another takes two.  Counts meet in distributed shared memory.
// Ranks come from counts in the order of pages or sequences, never from who is first, so results do not depend on timing.
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
constexpr int ROW_WARPS = 8;   // warps that share a sequence's row of the table, at most

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

// what all three have in common
struct Pages {
    const int32_t* lens;
    const int32_t* table;
    int batch, max_pages, num_pages, capacity;
    int row_warps;   // warps to a row
    FastDiv page;
    __device__ __forceinline__ int length(int b) const { return min(max(ld_s32(lens + b), 0), capacity); }
    __device__ __forceinline__ int pages_of(int n) const { return n > 0 ? (int)page.div((uint32_t)n - 1u) + 1 : 0; }
    __device__ __forceinline__ bool inside(int p) const { return (uint32_t)p < (uint32_t)num_pages; }
    // entry i of a ring from place `from` on; from and i are below num_pages
    __device__ __forceinline__ int ring_at(int from, int i) const {
        const uint32_t at = (uint32_t)from + (uint32_t)i;
        return (int)(at < (uint32_t)num_pages ? at : at - (uint32_t)num_pages);
    }
    // f(b, i, n): row b by n warps, of which this is the i-th
    template <class F>
    __device__ __forceinline__ void each_row(F&& f) const {
        const long long items = (long long)batch * row_warps;
        for (long long item = (long long)cluster_rank() * WARPS + (threadIdx.x >> 5); item < items; item += ALL_WARPS) f((int)(item / row_warps), (int)(item % row_warps), row_warps);
    }
    // f(p, valid): all pages, those of a warp one behind another, a warp's 32 at a time
    template <class F>
    __device__ __forceinline__ void each_page(F&& f) const {
        const long long per = ((long long)num_pages + ALL_THREADS - 1) / ALL_THREADS * 32;   // of a warp
        const long long first = (long long)(cluster_rank() * WARPS + (threadIdx.x >> 5)) * per;
        const int end = (int)min(first + per, (long long)num_pages);
        for (long long p0 = first; p0 < end; p0 += 32) {
            const int p = (int)p0 + (threadIdx.x & 31);
            f(p, p < end);
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
        for (int p = cluster_rank() * THREADS + threadIdx.x; p < a.num_pages; p += ALL_THREADS) to[p] = ld_s32(from + p);
}
__device__ __forceinline__ int gone_of(const int32_t* gone, int b) { return gone ? max(ld_s32(gone + b), 0) : 0; }

// ------------------------------------------------------------------------------------------------------------------- fork
struct Fork : Pages {
    const int32_t *parent, *keep, *ring, *state, *shares, *gone;
    int32_t *table_out, *lens_out, *state_out, *shares_out, *gone_out, *taken, *copy_from, *copy_to, *copies;
    int sink_pages;
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
    const int run = (a.batch + ALL_THREADS - 1) / ALL_THREADS;
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
            if (part && (int)full >= a.sink_pages && (int)full < gone_of(a.gone, p)) n = -1;   // its last page is not there any more
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
    // ---- the pages that are shared
    a.each_row([&](int b, int i, int n) {
        const int full = (int)a.page.div((uint32_t)ld_s32(a.taken + b));
        if (full == 0) return;
        const int p = ld_s32(a.parent + b), gone = gone_of(a.gone, p);
        const int32_t* from = a.table + (size_t)p * a.max_pages;
        int32_t* to = a.table_out + (size_t)b * a.max_pages;
        for (int j = 32 * i + lane; j < full; j += 32 * n) {
            if (j >= a.sink_pages && j < gone) continue;
            const int page = ld_s32(from + j);
            to[j] = page;
            if (a.inside(page)) atomicAdd(a.shares_out + page, 1);
        }
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
    __device__ __forceinline__ Cut(const Release& a, int b) {
        const int n = a.length(b);
        after = a.keep ? min(n, max(ld_s32(a.keep + b), 0)) : n;
        held = a.pages_of(n);
        gone = gone_of(a.gone, b);
        held_after = a.pages_of(after);
        const int passed = a.window && after >= a.window ? (int)a.page.div((uint32_t)(after - a.window) + 1u) : 0;   // the next token sees keys from after + 1 - window on
        left = min(max(gone, passed), held_after);
    }
};

// A page that nobody has any more has less than zero sharers.
__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__(THREADS, 1) kv_page_release_kernel(const Release a) {
    __shared__ int sh[1][WARPS + CTAS];
    const int rank = cluster_rank(), lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    const Ring ring(a.state, a.num_pages);
    if (a.shares != a.shares_out) {
        copy_shares(a, a.shares, a.shares_out);
        cluster_sync();
    }
    a.each_row([&](int b, int i, int n) {
        const Cut c(a, b);
        const int32_t* row = a.table + (size_t)b * a.max_pages;
        auto give = [&](int from, int to) {
            for (int j = from + 32 * i + lane; j < to; j += 32 * n) {
                const int page = ld_s32(row + j);
                if (a.inside(page)) atomicSub(a.shares_out + page, 1);
            }
        };
        // had: [0, sink_pages) and [gone, held); has: [0, sink_pages) and [left, held_after)
        give(c.held_after, min(a.sink_pages, c.held));
        const int from = max(c.gone, a.sink_pages);
        give(from, c.left);
        give(max(from, c.held_after), c.held);
    });
    cluster_sync();
    int mine = 0;
    a.each_page([&](int p, bool valid) { mine += __popc(__ballot_sync(0xffffffffu, valid && __ldcg(a.shares_out + p) < 0)); });
    const Before all = cluster_sum(mine, sh);
    int at = ring.count + all.warp;
    a.each_page([&](int p, bool valid) {
        const bool free = valid && __ldcg(a.shares_out + p) < 0;
        const uint32_t votes = __ballot_sync(0xffffffffu, free);
        if (free) {
            const int i = at + lanes_below(votes);
            if (i < a.num_pages) a.ring[a.ring_at(ring.head, i)] = p;   // a ring holds all pages
            a.shares_out[p] = 0;
        }
        at += __popc(votes);
    });
    for (int b = rank * THREADS + threadIdx.x; b < a.batch; b += ALL_THREADS) {
        const Cut c(a, b);
        a.lens_out[b] = c.after;
        if (a.gone_out) a.gone_out[b] = c.left;
    }
    if (rank == 0 && threadIdx.x == 0) {
        a.state_out[0] = ring.head;
        a.state_out[1] = min(ring.count + all.total, a.num_pages);
    }
}

// ---------------------------------------------------------------------------------------------------------------- compact
struct Compact : Pages {
    const int32_t *ring, *state, *shares;
    int32_t *table_out, *ring_out, *state_out, *shares_out, *moved_to, *copy_from, *copy_to, *copies;
};

__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__(THREADS, 1) kv_page_compact_kernel(const Compact a) {
    __shared__ int sh[2][WARPS + CTAS];
    const int rank = cluster_rank(), lane = threadIdx.x & 31, thread = rank * THREADS + threadIdx.x;
    pdl_wait();
    pdl_trigger();
    const Ring ring(a.state, a.num_pages);
    for (int p = thread; p < a.num_pages; p += ALL_THREADS) a.moved_to[p] = 0;
    cluster_sync();
    for (int i = thread; i < ring.count; i += ALL_THREADS) {
        const int p = ld_s32(a.ring + a.ring_at(ring.head, i));
        if (a.inside(p)) a.moved_to[p] = -1;   // free
    }
    cluster_sync();
    // ---- the used pages are to be those below `used`: the others of them move to the free ones there, in order
    auto is_used = [&](int p, bool valid) { return valid && __ldcg(a.moved_to + p) == 0; };
    int mine = 0;
    a.each_page([&](int p, bool valid) { mine += __popc(__ballot_sync(0xffffffffu, is_used(p, valid))); });
    const Before of_used = cluster_sum(mine, &sh[0]);
    const int used = of_used.total;
    mine = 0;
    a.each_page([&](int p, bool valid) { mine += __popc(__ballot_sync(0xffffffffu, is_used(p, valid) && p >= used)); });
    const Before of_movers = cluster_sum(mine, &sh[1]);
    int movers = of_movers.warp, below = of_used.warp;
    a.each_page([&](int p, bool valid) {
        const bool u = is_used(p, valid), moves = u && p >= used;
        const uint32_t votes = __ballot_sync(0xffffffffu, u), moving = __ballot_sync(0xffffffffu, moves);
        if (moves) a.copy_from[movers + lanes_below(moving)] = p;
        if (valid && !u && p < used) a.copy_to[p - (below + lanes_below(votes))] = p;
        below += __popc(votes);
        movers += __popc(moving);
    });
    cluster_sync();
    movers = of_movers.warp;
    a.each_page([&](int p, bool valid) {
        const bool u = is_used(p, valid), moves = u && p >= used;
        const uint32_t moving = __ballot_sync(0xffffffffu, moves);
        if (u) {
            const int to = moves ? __ldcg(a.copy_to + movers + lanes_below(moving)) : p;
            a.moved_to[p] = to;
            a.shares_out[to] = ld_s32(a.shares + p);
        }
        if (valid && p >= used) a.shares_out[p] = 0;
        movers += __popc(moving);
    });
    cluster_sync();
    a.each_row([&](int b, int i, int n) {
        const int held = a.pages_of(a.length(b));
        const size_t row = (size_t)b * a.max_pages;
        for (int j = 32 * i + lane; j < held; j += 32 * n) {
            const int p = ld_s32(a.table + row + j);
            a.table_out[row + j] = a.inside(p) ? __ldcg(a.moved_to + p) : -1;
        }
    });
    for (int i = thread; i < a.num_pages; i += ALL_THREADS) a.ring_out[i] = i < a.num_pages - used ? used + i : -1;
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
// Bound by memory.
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
    a.row_warps = (max_pages + 31) / 32;
    if (a.row_warps > ROW_WARPS) a.row_warps = ROW_WARPS;
    return true;
}
int pages_behind(int tokens, int page_size) { return (int)(((long long)tokens + page_size - 1) / page_size); }

}  // namespace

extern "C" int kv_page_fork(const kv_page_fork_args_t* g) {
    if (!g || !g->lens || !g->parent || !g->block_table || !g->ring || !g->ring_state || !g->shares || !g->lens_out || !g->ring_state_out || !g->shares_out || !g->taken ||
        !g->copy_from || !g->copy_to || !g->copies || !g->gone != !g->gone_out || g->sinks < 0)
        return (int)cudaErrorInvalidValue;
    if (!words({g->lens, g->parent, g->keep, g->block_table, g->ring, g->ring_state, g->shares, g->gone, g->lens_out, g->ring_state_out, g->shares_out, g->gone_out, g->taken,
                g->copy_from, g->copy_to, g->copies}))
        return (int)cudaErrorInvalidValue;
    Fork a;
    if (!fill(a, g->lens, g->block_table, g->batch, g->max_pages_per_seq, g->page_size, g->num_pages)) return (int)cudaErrorInvalidValue;
    a.parent = g->parent; a.keep = g->keep; a.ring = g->ring; a.state = g->ring_state; a.shares = g->shares; a.gone = g->gone;
    a.table_out = g->block_table; a.lens_out = g->lens_out; a.state_out = g->ring_state_out; a.shares_out = g->shares_out; a.gone_out = g->gone_out; a.taken = g->taken;
    a.copy_from = g->copy_from; a.copy_to = g->copy_to; a.copies = g->copies;
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
