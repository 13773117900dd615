// kv_pages_sm100.cu — the pages and places of a step of a paged KV cache, planned on the GPU (kv_page_plan, include/fp8_block.h).
//
// Three running sums over the sequences say everything: of the new tokens (where a sequence's rows start), of the pages that sequences need, and of the pages that
// they give back.  Every CTA forms them for itself (a batch is a few thousand numbers, which L2 serves), then takes tiles of the step's rows and of the returned
// pages.  A tile finds the sequence of each of its rows by marking where sequences start and a running maximum of the marks.
//
// What a CTA reads, no CTA writes: new pages come from the front of the ring and returned ones go behind its end, only new entries of the table are written, and the
// lengths and the ring's state, which may be updated in place, are written by the CTA that finishes last.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/fp8_block.h"
#include "pdl.cuh"
#include "row_items.cuh"

namespace {

using namespace sm100;

constexpr int CTAS_PER_SM = 4;

struct Plan {
    const int32_t *lens, *fresh;
    int32_t *table, *ring, *state, *lens_out, *state_out, *taken, *starts, *positions, *slots;
    int batch, max_pages, page_size, num_pages, rows, per_seq;
    int capacity;   // of a sequence, in tokens
    int run;        // sequences of a thread: thread i has those from i * run on
    FastDiv page;
    __device__ __forceinline__ int pages_of(int n) const { return n > 0 ? (int)page.div((uint32_t)n - 1u) + 1 : 0; }
    // entry i of the ring from place `from` on; from and i are below num_pages
    __device__ __forceinline__ int32_t* ring_at(int from, long long i) const {
        const uint32_t at = (uint32_t)from + (uint32_t)i;
        return ring + (at < (uint32_t)num_pages ? at : at - (uint32_t)num_pages);
    }
};

struct Sums {
    long long rows, need, back;
};

// what sequence b wants
struct Sequence {
    int len, fresh, held;
    bool ends;
    __device__ __forceinline__ Sequence(const Plan& a, int b) {
        len = min(max(ld_s32(a.lens + b), 0), a.capacity);
        fresh = ld_s32(a.fresh + b);
        ends = fresh < 0;
        fresh = max(fresh, 0);
        held = a.pages_of(len);
    }
    // pages that it needs, given where its rows start; 0 and fits = false where it cannot be taken whatever the ring has
    __device__ __forceinline__ int need(const Plan& a, long long start, bool& fits) const {
        fits = fresh > 0 && (long long)len + fresh <= a.capacity && (a.per_seq ? fresh <= a.per_seq : start + fresh <= a.rows);
        return fits ? a.pages_of(len + fresh) - held : 0;
    }
};

// exclusive sums over the block's threads in order, and the total
template <int THREADS>
__device__ __forceinline__ long long block_sum(long long x, long long& total, long long* sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long incl = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    __syncthreads();   // sh may still be read
    if (lane == 31) sh[warp] = incl;
    __syncthreads();
    long long before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) {
        if (w < warp) before += sh[w];
        total += sh[w];
    }
    return before + incl - x;
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) kv_page_plan_kernel(const Plan a) {
    __shared__ long long sh[THREADS / 32];
    __shared__ int s_mark[THREADS];        // sequence whose first row in the tile this is, or -1
    __shared__ long long s_start[THREADS]; // its first row of all
    __shared__ long long s_base[THREADS];  // and its first new page's place in the ring
    __shared__ int s_top[THREADS / 32];
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    pdl_trigger();
    const int head = (int)((uint32_t)max(ld_s32(a.state), 0) % (uint32_t)a.num_pages), count = min(max(ld_s32(a.state + 1), 0), a.num_pages);
    const int b_begin = min(tid * a.run, a.batch), b_end = min(b_begin + a.run, a.batch);

    // ---- where this thread's sequences start
    Sums mine{0, 0, 0}, total;
    for (int b = b_begin; b < b_end; b++) {
        const Sequence s(a, b);
        mine.rows += min((long long)s.fresh, (long long)a.rows + 1);   // one that is longer than the step's rows keeps those behind it out, too
        mine.back += s.ends ? s.held : 0;
    }
    Sums first;
    first.rows = block_sum<THREADS>(mine.rows, total.rows, sh);
    first.back = block_sum<THREADS>(mine.back, total.back, sh);
    // one sequence at a time, with what lies before it
    auto each = [&](long long need_before, auto&& f) {
        Sums at = first;
        at.need = need_before;
        for (int b = b_begin; b < b_end; b++) {
            const Sequence s(a, b);
            const long long start = a.per_seq ? (long long)b * a.per_seq : at.rows;
            bool fits;
            const int need = s.need(a, start, fits);
            f(b, s, start, need, fits && (need == 0 || at.need + need <= count), at);
            at.rows += min((long long)s.fresh, (long long)a.rows + 1);
            at.need += need;
            at.back += s.ends ? s.held : 0;
        }
    };
    each(0, [&](int, const Sequence&, long long, int need, bool, const Sums&) { mine.need += need; });
    first.need = block_sum<THREADS>(mine.need, total.need, sh);
    const long long back = min(total.back, (long long)a.num_pages - count);   // a ring holds num_pages

    // ---- this CTA's share of what is one number a sequence
    long long used_mine = 0;
    each(first.need, [&](int b, const Sequence& s, long long start, int need, bool served, const Sums&) {
        used_mine += served ? need : 0;
        if (b % gridDim.x == blockIdx.x) {
            a.taken[b] = served ? s.fresh : 0;
            a.starts[b] = (int)min(start, (long long)a.rows);
        }
    });
    if (blockIdx.x == 0 && tid == 0) a.starts[a.batch] = (int)min(a.per_seq ? (long long)a.batch * a.per_seq : total.rows, (long long)a.rows);

    // the mark that a row of the tile belongs to: the last one at or before it, or -1
    auto owner = [&]() -> int {
        int at = s_mark[tid] >= 0 ? tid : -1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= o) at = max(at, y);
        }
        if (lane == 31) s_top[warp] = at;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 32; w++)
            if (w < warp) at = max(at, s_top[w]);
        return at;
    };

    // ---- tiles of the step's rows
    for (long long r0 = (long long)blockIdx.x * THREADS; r0 < a.rows; r0 += (long long)gridDim.x * THREADS) {
        __syncthreads();
        s_mark[tid] = -1;
        __syncthreads();
        each(first.need, [&](int b, const Sequence& s, long long start, int, bool served, const Sums& at) {
            if (served && start < r0 + THREADS && start + s.fresh > r0) {   // those that are taken have rows of their own
                const int i = (int)(max(start, r0) - r0);
                s_mark[i] = b;
                s_start[i] = start;
                s_base[i] = at.need;
            }
        });
        __syncthreads();
        const int o = owner();
        const long long row = r0 + tid;
        if (row < a.rows) {
            int position = -1, slot = -1;
            if (o >= 0) {
                const int b = s_mark[o];
                const Sequence s(a, b);
                const long long k = row - s_start[o];
                if (k < s.fresh) {
                    position = s.len + (int)k;
                    uint32_t j, place;
                    a.page.divmod((uint32_t)position, j, place);
                    int32_t* entry = a.table + (size_t)b * a.max_pages + j;
                    int pg;
                    if ((int)j < s.held) {
                        pg = ld_s32(entry);
                    } else {
                        pg = ld_s32(a.ring_at(head, s_base[o] + j - s.held));
                        if (place == 0) *entry = pg;   // a new page's first token
                    }
                    if (pg >= 0 && pg < a.num_pages) slot = pg * a.page_size + (int)place;
                }
            }
            a.positions[row] = position;
            a.slots[row] = slot;
        }
    }

    // ---- tiles of the returned pages
    for (long long r0 = (long long)blockIdx.x * THREADS; r0 < back; r0 += (long long)gridDim.x * THREADS) {
        __syncthreads();
        s_mark[tid] = -1;
        __syncthreads();
        each(first.need, [&](int b, const Sequence& s, long long, int, bool, const Sums& at) {
            if (s.ends && s.held > 0 && at.back < r0 + THREADS && at.back + s.held > r0) {
                const int i = (int)(max(at.back, r0) - r0);
                s_mark[i] = b;
                s_start[i] = at.back;
            }
        });
        __syncthreads();
        const int o = owner();
        const long long r = r0 + tid;
        if (r < back && o >= 0)
            *a.ring_at(head, count + r) = ld_s32(a.table + (size_t)s_mark[o] * a.max_pages + (r - s_start[o]));
    }

    // ---- lengths and state, which other CTAs may still have to read: by the last one
    long long used;
    block_sum<THREADS>(used_mine, used, sh);
    if (gridDim.x > 1) {
        __threadfence();
        __syncthreads();
        if (tid == 0) s_last = atomicAdd(reinterpret_cast<unsigned int*>(a.state + 2), 1u) == gridDim.x - 1;
        __syncthreads();
        if (!s_last) return;
        __threadfence();
        if (tid == 0) a.state[2] = 0;
    }
    each(first.need, [&](int b, const Sequence& s, long long, int, bool served, const Sums&) { a.lens_out[b] = s.ends ? 0 : s.len + (served ? s.fresh : 0); });
    if (tid == 0) {
        a.state_out[0] = (int)((head + used) % a.num_pages);
        a.state_out[1] = (int)(count - used + back);
    }
}

}  // namespace

extern "C" int kv_page_plan(const kv_page_plan_args_t* g) {
    if (!g || !g->lens || !g->fresh || !g->block_table || !g->ring || !g->ring_state || !g->lens_out || !g->ring_state_out || !g->taken || !g->starts) return (int)cudaErrorInvalidValue;
    if (g->batch < 0 || g->rows < 0 || g->max_pages_per_seq <= 0 || g->page_size <= 0 || g->num_pages <= 0 || g->tokens_per_seq < 0) return (int)cudaErrorInvalidValue;
    if (g->rows > 0 && (!g->positions || !g->slots)) return (int)cudaErrorInvalidValue;
    if ((long long)g->page_size * g->max_pages_per_seq > 0x7fffffffLL || (long long)g->page_size * g->num_pages > 0x7fffffffLL ||
        (long long)g->batch * g->tokens_per_seq > g->rows)
        return (int)cudaErrorInvalidValue;
    for (const void* p : {(const void*)g->lens, (const void*)g->fresh, (const void*)g->block_table, (const void*)g->ring, (const void*)g->ring_state, (const void*)g->lens_out,
                          (const void*)g->ring_state_out, (const void*)g->taken, (const void*)g->starts, (const void*)g->positions, (const void*)g->slots})
        if (reinterpret_cast<uintptr_t>(p) & 3) return (int)cudaErrorInvalidValue;
    Plan a;
    a.lens = g->lens; a.fresh = g->fresh; a.table = g->block_table; a.ring = g->ring; a.state = g->ring_state; a.lens_out = g->lens_out;
    a.state_out = g->ring_state_out; a.taken = g->taken; a.starts = g->starts; a.positions = g->positions; a.slots = g->slots;
    a.batch = g->batch; a.max_pages = g->max_pages_per_seq; a.page_size = g->page_size; a.num_pages = g->num_pages; a.rows = g->rows; a.per_seq = g->tokens_per_seq;
    a.capacity = g->page_size * g->max_pages_per_seq;
    a.page = FastDiv((uint32_t)g->page_size);
    constexpr int THREADS = 512;
    a.run = (g->batch + THREADS - 1) / THREADS;
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    long long grid = ((long long)g->rows + THREADS - 1) / THREADS;
    if (grid > (long long)sms * CTAS_PER_SM) grid = (long long)sms * CTAS_PER_SM;
    return (int)launch_pdl(kv_page_plan_kernel<THREADS>, dim3((unsigned)(grid > 0 ? grid : 1)), dim3(THREADS), 0, (cudaStream_t)g->stream, a);
}
