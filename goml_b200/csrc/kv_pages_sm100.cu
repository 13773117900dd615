// kv_pages_sm100.cu — the pages and places of a step of a paged KV cache, planned on the GPU (kv_page_plan, include/fp8_block.h).
//
// Three running sums over the sequences say everything: of the new tokens (where a sequence's rows start), of the pages that sequences need, and of the pages that
// they give back.  Every CTA forms them for itself (a thread has up to four sequences side by side, in registers), then takes tiles of the step's rows and of the returned pages.  A tile finds the sequence of each of its rows by marking where sequences start and a running maximum of the marks.
//
// What a CTA reads, no CTA writes: new pages come from the front of the ring and returned ones go behind its end, only new entries of the table are written, and the
// lengths and the ring's state, which may be updated in place, are written by the CTA that is last to have read them.
//
// Bound by latency: a chain of lengths, exchanges across the CTA, table entries and ring.  8 sequences 3.4 us, 192 with 16384 rows 5.3, 1000 with 60000 6.6, 4096 with 300000 11.0.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/fp8_block.h"
#include "pdl.cuh"
#include "row_items.cuh"

namespace {

using namespace sm100;

struct Plan {
    const int32_t *lens, *fresh;
    int32_t *table, *ring, *state, *lens_out, *state_out, *taken, *starts, *positions, *slots;
    int batch, max_pages, page_size, num_pages, rows, per_seq;
    int capacity;   // of a sequence, in tokens
    int run;        // sequences of a thread: thread i has those from i * run on
    bool wide;      // positions and slots are 8-byte aligned
    FastDiv page;
    __device__ __forceinline__ int pages_of(int n) const { return n > 0 ? (int)page.div((uint32_t)n - 1u) + 1 : 0; }
    // entry i of the ring from place `from` on; from and i are below num_pages
    __device__ __forceinline__ int32_t* ring_at(int from, int i) const {
        const uint32_t at = (uint32_t)from + (uint32_t)i;
        return ring + (at < (uint32_t)num_pages ? at : at - (uint32_t)num_pages);
    }
};

// Sums stop at 2^31 - 1, which is past the last row, page and ring entry: the same whatever the order.
__device__ __forceinline__ int plus(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, 0x7fffffffu); }
struct Sums {
    int rows, need, back;
};

// what a sequence wants
struct Sequence {
    int len, fresh, held;
    bool ends;
    __device__ __forceinline__ Sequence(const Plan& a, int n, int f) {
        len = min(max(n, 0), a.capacity);
        ends = f < 0;
        fresh = max(f, 0);
        held = a.pages_of(len);
    }
    // pages that it needs, given where its rows start; 0 and fits = false where it cannot be taken whatever the ring has
    __device__ __forceinline__ int need(const Plan& a, int start, bool& fits) const {
        fits = fresh > 0 && (long long)len + fresh <= a.capacity && (a.per_seq ? fresh <= a.per_seq : (long long)start + fresh <= a.rows);
        return fits ? a.pages_of(len + fresh) - held : 0;
    }
};

// exclusive sums over the block's threads in order, and the total
template <int THREADS, int N>
__device__ __forceinline__ void block_sum(int (&x)[N], int (&total)[N], int (*sh)[N]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl[N];
#pragma unroll
    for (int k = 0; k < N; k++) incl[k] = x[k];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int y = __shfl_up_sync(0xffffffffu, incl[k], o);
            if (lane >= o) incl[k] = plus(incl[k], y);
        }
    __syncthreads();   // sh may still be read
    if (lane == 31)
#pragma unroll
        for (int k = 0; k < N; k++) sh[warp][k] = incl[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; k++) {
        // every warp adds the warps' sums up for itself: few one by one, many by exchanges (of four 0.3 us slower, of 32 3.3 us faster)
        int before = 0;
        total[k] = 0;
        if (THREADS <= 128) {
#pragma unroll
            for (int w = 0; w < THREADS / 32; w++) {
                if (w < warp) before = plus(before, sh[w][k]);
                total[k] = plus(total[k], sh[w][k]);
            }
        } else {
            int warps = lane < THREADS / 32 ? sh[lane][k] : 0;
#pragma unroll
            for (int o = 1; o < THREADS / 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, warps, o);
                if (lane >= o) warps = plus(warps, y);
            }
            total[k] = __shfl_sync(0xffffffffu, warps, THREADS / 32 - 1);
            if (warp) before = __shfl_sync(0xffffffffu, warps, warp - 1);
        }
        const int y = __shfl_up_sync(0xffffffffu, incl[k], 1);
        x[k] = lane ? plus(before, y) : before;
    }
}

// RUN: sequences of a thread, kept in registers; 0: any number, read where they are looked at
// TILE: rows of a thread in a tile
template <int THREADS, int RUN, int TILE>
__global__ void __launch_bounds__(THREADS) kv_page_plan_kernel(const Plan a) {
    constexpr int ROWS = THREADS * TILE;
    __shared__ int sh2[THREADS / 32][2], sh1[THREADS / 32][1];
    // of the sequence whose first row in the tile this is: itself (-1: none), its first row of all, length, new tokens and first new page's place in the ring
    __shared__ int s_mark[ROWS], s_start[ROWS], s_len[ROWS], s_fresh[ROWS], s_base[ROWS];
    __shared__ int s_top[THREADS / 32];
    __shared__ int s_state[2], s_used, s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    pdl_trigger();
    const int run = RUN ? RUN : a.run, b_begin = min(tid * run, a.batch), b_end = min(b_begin + run, a.batch);
    int len_of[RUN ? RUN : 1], fresh_of[RUN ? RUN : 1];
    if (RUN) {
#pragma unroll
        for (int i = 0; i < RUN; i++) {
            len_of[i] = fresh_of[i] = 0;
            if (b_begin + i < b_end) {
                len_of[i] = __ldcg(a.lens + b_begin + i);
                fresh_of[i] = __ldcg(a.fresh + b_begin + i);
            }
        }
    }
    if (tid < 2) s_state[tid] = ld_s32(a.state + tid);
    if (tid == 0) s_used = s_last = 0;
    auto each_sequence = [&](auto&& f) {
        if (RUN) {
#pragma unroll
            for (int i = 0; i < RUN; i++)
                if (b_begin + i < b_end) f(b_begin + i, Sequence(a, len_of[i], fresh_of[i]));
        } else {
            for (int b = b_begin; b < b_end; b++) f(b, Sequence(a, __ldcg(a.lens + b), __ldcg(a.fresh + b)));
        }
    };

    // ---- where this thread's sequences start
    Sums first;
    int rows_total, back_total;
    {
        int x[2] = {0, 0}, total[2];
        each_sequence([&](int, const Sequence& s) {
            x[0] = plus(x[0], s.fresh);
            x[1] = plus(x[1], s.ends ? s.held : 0);
        });
        block_sum<THREADS, 2>(x, total, sh2);   // (the ring's state is there behind it, too)
        first.rows = x[0];
        first.back = x[1];
        rows_total = total[0];
        back_total = total[1];
    }
    const int head = (int)((uint32_t)max(s_state[0], 0) % (uint32_t)a.num_pages), count = min(max(s_state[1], 0), a.num_pages);
    // Whether this CTA is the last to have read what may be updated in place
    auto arrive = [&] {
        if (tid != 0) return;
        bool last = true;
        if (gridDim.x > 1) {
            __threadfence();
            last = atomicAdd(reinterpret_cast<unsigned int*>(a.state + 2), 1u) == gridDim.x - 1;
            if (last) a.state[2] = 0;
        }
        s_last = last;
    };
    if (RUN) arrive();
    // one sequence at a time, with what lies before it
    auto each = [&](int need_before, auto&& f) {
        Sums at = first;
        at.need = need_before;
        each_sequence([&](int b, const Sequence& s) {
            const int start = a.per_seq ? b * a.per_seq : at.rows;
            bool fits;
            const int need = s.need(a, start, fits);
            f(b, s, start, need, fits && (need == 0 || plus(at.need, need) <= count), at);
            at.rows = plus(at.rows, s.fresh);
            at.need = plus(at.need, need);
            at.back = plus(at.back, s.ends ? s.held : 0);
        });
    };
    {
        int x[1] = {0}, total[1];
        each(0, [&](int, const Sequence&, int, int need, bool, const Sums&) { x[0] = plus(x[0], need); });
        block_sum<THREADS, 1>(x, total, sh1);
        first.need = x[0];
    }
    const int back = min(back_total, a.num_pages - count);   // a ring holds num_pages

    // the marks that a thread's rows of the tile belong to: the last one at or before each, or -1
    auto owners = [&](int (&of)[TILE]) {
        int at = -1;
#pragma unroll
        for (int i = 0; i < TILE; i++) {
            if (s_mark[TILE * tid + i] >= 0) at = TILE * tid + i;
            of[i] = at;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= o) at = max(at, y);
        }
        if (lane == 31) s_top[warp] = at;
        __syncthreads();
        int before = __shfl_up_sync(0xffffffffu, at, 1);
        before = max(lane ? before : -1, __reduce_max_sync(0xffffffffu, lane < warp ? s_top[lane] : -1));
#pragma unroll
        for (int i = 0; i < TILE; i++) of[i] = max(of[i], before);
    };
    auto clear_marks = [&] {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TILE; i++) s_mark[THREADS * i + tid] = -1;
        __syncthreads();
    };

    // ---- tiles of the step's rows, and with the first one this CTA's share of what is one number a sequence: those of some of its warps
    const bool shares = warp % (int)gridDim.x == (int)blockIdx.x % (THREADS / 32) && (int)blockIdx.x < THREADS / 32;
    long long tile = (long long)blockIdx.x * ROWS;
    bool first_tile = true;
    do {
        const int r0 = (int)min(tile, 0x7fffffffLL);
        clear_marks();
        int used_mine = 0;
        each(first.need, [&](int b, const Sequence& s, int start, int need, bool served, const Sums& at) {
            if (first_tile) {
                if (served && need) used_mine = at.need + need;
                if (shares) {
                    a.taken[b] = served ? s.fresh : 0;
                    a.starts[b] = min(start, a.rows);
                }
                if (RUN && s_last) a.lens_out[b] = s.ends ? 0 : s.len + (served ? s.fresh : 0);
            }
            if (served && start - r0 < ROWS && s.fresh > r0 - start) {   // those that are taken have rows of their own
                const int i = max(start - r0, 0);
                s_mark[i] = b;
                s_start[i] = start;
                s_len[i] = s.len;
                s_fresh[i] = s.fresh;
                s_base[i] = at.need;
            }
        });
        if (used_mine) atomicMax(&s_used, used_mine);
        first_tile = false;
        if (tile >= a.rows) break;   // a step without rows
        __syncthreads();
        int of[TILE], position[TILE], slot[TILE];
        owners(of);
#pragma unroll
        for (int i = 0; i < TILE; i++) {
            const int o = of[i], k = o < 0 ? 0 : r0 + TILE * tid + i - s_start[o];
            position[i] = slot[i] = -1;
            if (o < 0 || k >= s_fresh[o] || TILE * tid + i >= a.rows - r0) continue;
            position[i] = s_len[o] + k;
            const int held = a.pages_of(s_len[o]);
            uint32_t j, place;
            a.page.divmod((uint32_t)position[i], j, place);
            int32_t* entry = a.table + (size_t)s_mark[o] * a.max_pages + j;
            const bool is_new = (int)j >= held;
            const int pg = __ldcg(is_new ? a.ring_at(head, s_base[o] + (int)j - held) : entry);
            if (is_new && place == 0) *entry = pg;   // a new page's first token
            if (pg >= 0 && pg < a.num_pages) slot[i] = pg * a.page_size + (int)place;
        }
        const long long row = tile + TILE * tid;
        if (TILE == 2 && a.wide && row + TILE <= a.rows) {
            *reinterpret_cast<int2*>(a.positions + row) = make_int2(position[0], position[TILE - 1]);
            *reinterpret_cast<int2*>(a.slots + row) = make_int2(slot[0], slot[TILE - 1]);
        } else {
#pragma unroll
            for (int i = 0; i < TILE; i++)
                if (row + i < a.rows) {
                    a.positions[row + i] = position[i];
                    a.slots[row + i] = slot[i];
                }
        }
        tile += (long long)gridDim.x * ROWS;
    } while (tile < a.rows);
    if (blockIdx.x == 0 && tid == 0) a.starts[a.batch] = min(a.per_seq ? a.batch * a.per_seq : rows_total, a.rows);

    // ---- tiles of the returned pages
    for (long long tile = (long long)blockIdx.x * ROWS; tile < back; tile += (long long)gridDim.x * ROWS) {
        const int r0 = (int)tile;
        clear_marks();
        each(first.need, [&](int b, const Sequence& s, int, int, bool, const Sums& at) {
            if (s.ends && s.held > 0 && at.back < back && at.back - r0 < ROWS && s.held > r0 - at.back) {
                const int i = max(at.back - r0, 0);
                s_mark[i] = b;
                s_start[i] = at.back;
            }
        });
        __syncthreads();
        int of[TILE];
        owners(of);
#pragma unroll
        for (int i = 0; i < TILE; i++) {
            const int o = of[i], r = TILE * tid + i;   // from r0 on
            if (o >= 0 && r < back - r0) *a.ring_at(head, count + r0 + r) = __ldcg(a.table + (size_t)s_mark[o] * a.max_pages + (r0 + r - s_start[o]));
        }
    }

    __syncthreads();
    if (!RUN) {
        arrive();
        __syncthreads();
        if (s_last) each(first.need, [&](int b, const Sequence& s, int, int, bool served, const Sums&) { a.lens_out[b] = s.ends ? 0 : s.len + (served ? s.fresh : 0); });
    }
    if (s_last && tid == 0) {
        a.state_out[0] = (int)(((uint32_t)head + (uint32_t)s_used) % (uint32_t)a.num_pages);
        a.state_out[1] = count - s_used + back;
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
    a.wide = ((reinterpret_cast<uintptr_t>(g->positions) | reinterpret_cast<uintptr_t>(g->slots)) & 7) == 0;
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const cudaStream_t s = (cudaStream_t)g->stream;
    auto run = [&](auto kernel, int threads, int tile) {
        const long long tiles = ((long long)g->rows + threads * tile - 1) / (threads * tile);
        a.run = (g->batch + threads - 1) / threads;
        return (int)launch_pdl(kernel, dim3((unsigned)(tiles < 1 ? 1 : tiles < sms ? tiles : sms)), dim3(threads), 0, s, a);
    };
    if (g->batch <= 128 && g->rows <= 128) return run(kv_page_plan_kernel<128, 1, 1>, 128, 1);
    if (g->batch <= 512 && g->rows <= sms * 512LL) return run(kv_page_plan_kernel<512, 1, 1>, 512, 1);
    // One row to a thread while the SMs have room for as many CTAs (1000 sequences, 60000 rows, one 6.6 us, two 7.6; 4096 with 300000 rows, of which that takes two rounds, 15.8 and 14.2
    // before the sums across warps were exchanges), and few threads for few sequences.
    const bool one_round = g->rows <= sms * 1024LL;
    if (g->batch <= 1024) return one_round ? run(kv_page_plan_kernel<1024, 1, 1>, 1024, 1) : run(kv_page_plan_kernel<1024, 1, 2>, 1024, 2);
    if (g->batch <= 4096) return one_round ? run(kv_page_plan_kernel<1024, 4, 1>, 1024, 1) : run(kv_page_plan_kernel<1024, 4, 2>, 1024, 2);
    return run(kv_page_plan_kernel<1024, 0, 2>, 1024, 2);
}
