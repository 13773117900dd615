// fa_decode_stream_sm100.cu — FP8 decode attention over a part of each sequence's keys (sm_100a): a window with the first tokens (fa_decode_window), or what a
// sequence has behind a shared prefix (the first kernel of fa_decode_shared).
//
// For one query the keys that it sees are two runs, [0, head) and [lo, len); the chunks of 64 keys that hold any of them, sinks first, are the sequence's line, and the lines
// of all pairs (sequence, kv head) one behind another are cut into equal pieces, one for every resident CTA.  Each byte is used once, 4 flops of the tensor cores
// for each query head that shares it: bound by memory.  So
//  * one warp of a CTA (the producer) walks the piece and keeps a ring of chunks full, with one tensor-map copy each for K and V (swizzled, so that fragments are read without
//    bank conflicts; rows past a cache's end and pages that the pool does not have arrive as zeros), across the ends of pairs.  What belongs to a chunk, masks and ends of pairs
//    among it, it writes beside it, so that
//  * four warps take 16 keys of every chunk each and look at nothing else: S^T = K Q^T (m16n8k32 on the codes), a running maximum that may lag by 2^6 (its rescaling is rare),
//    P in fp16, O^T += V^T P^T (m16n8k16 on V converted in registers).
//  * The warps' states of a pair meet in shared memory, where a sixth warp adds them up while the next pair is attended to.  Pieces of a pair that is cut meet in a workspace, where the CTA that is last adds them up in order: results
//    do not depend on timing.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>
#include <initializer_list>

#include "../../include/fa_sm120.h"
#include "fa_decode_mma.cuh"
#include "fa_decode_stream.h"
#include "fa_scratch_call.h"
#include "pdl.cuh"
#include "row_items.cuh"
#include "sm100_ptx.cuh"
#include "tmap.cuh"

namespace fa_sm100 {

namespace {

using namespace sm100;

constexpr int CHUNK = 64;   // keys (page sizes are multiples of it)
constexpr int CONSUMERS = 4, PRODUCER = 4, FINISHER = 5, THREADS = 32 * 6;
constexpr float LAG = 6.0f;   // log2 units
enum : uint32_t { ST_STREAM_LOAD = 0x241, ST_STREAM_USE = 0x242, ST_STREAM_MEET = 0x243, ST_STREAM_FINISH = 0x244 };

template <int D, int NQ>
struct Cfg {
    // Few CTAs with many chunks on their way each: with three to an SM and three chunks each, 128 sequences of 4100 keys, 8 kv heads of 128, 199 us, now 174; 64 of 4096, 32
    // heads, 376, now 323.
    static constexpr int CTAS = 2;                     // resident on an SM
    static constexpr int STAGES = D == 128 ? NQ == 1 ? 4 : 4 : 8;
    static constexpr int BUFFERS = NQ == 1 ? 2 : 1;    // of the warps' states on their way to a pair's sum
    static constexpr int ROWS = 8 * NQ;                // query columns
    static constexpr int PITCH = D + 4;                // floats of a row of the merge buffer
    static constexpr int TILE = CHUNK * D;             // bytes of a chunk of K or V
    static constexpr int KW = D / 16;                  // words of a lane's share of a K row
    static constexpr int MT = D / 16;                  // 16-row tiles of O^T
    static constexpr int VW = D / 32;                  // words of a lane's share of a V row
    static constexpr int OFF_V = STAGES * TILE;
    static constexpr int OFF_Q = 2 * STAGES * TILE;
    static constexpr int OFF_INFO = OFF_Q + STAGES * ROWS * D;
    static constexpr int OFF_BAR = OFF_INFO + STAGES * 48;
    static constexpr int OFF_FLAG = OFF_BAR + 16 * STAGES + 16 * BUFFERS + 8;   // behind two barriers a stage and a buffer and one of the consumers
    static constexpr int OFF_PAIR = OFF_FLAG + 8;      // [BUFFERS]: the pair of a buffer
    static constexpr int OFF_O = (OFF_PAIR + 4 * BUFFERS + 127) & -128;
    static constexpr int O_BYTES = CONSUMERS * ROWS * PITCH * 4, ML_BYTES = CONSUMERS * ROWS * 8;
    static constexpr int OFF_ML = OFF_O + BUFFERS * O_BYTES;
    static constexpr int SMEM = OFF_ML + BUFFERS * ML_BYTES + 1024;   // and what aligns it
    static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "all are resident");
};

struct Params {
    const uint8_t* q;
    __half* o;
    float* lse;
    const int* seq_lens;
    const int* shared_lens;
    int batch, hkv, group, s_max, seq_len, window, sinks;
    float scale_log2, v_descale;
    const float *sq, *sk, *sv;
    const int* block_table;   // nullptr: contiguous
    int max_pages, num_pages, page_size;
    FastDiv page;
    float *ws_o, *ws_ml;      // two slots a CTA: [slot][rows][D], [slot][rows][2]
    uint32_t* arrivals;       // [batch * hkv]
    float *own_o, *own_ml;    // shared_lens: the states [batch * q heads][D], [..][2], in the place of O and LSE
    uint32_t* status;
};

// The keys that a sequence sees, as chunks: `head` keys in the first `head_chunks`, then those from chunk head_chunks + skip on.
struct Span {
    int len, lo, head, head_chunks, skip, n;
    __device__ __forceinline__ Span(const Params& p, int length, int shared) {
        len = length;
        if (p.shared_lens) {
            lo = min(max(shared, 0), len);
            head = 0;
        } else {
            lo = p.window > 0 && len > p.window ? len - p.window : 0;
            head = min(p.sinks, lo);
            if (head == lo) lo = head = 0;
        }
        // (of nothing behind the prefix, the chunk of the last key: every pair has one, and with it a state)
        const int first = max(min(lo, len - 1), 0) / CHUNK;
        head_chunks = (head + CHUNK - 1) / CHUNK;
        const int from = max(first, head_chunks);
        skip = from - head_chunks;
        n = len > 0 ? head_chunks + max((len - 1) / CHUNK + 1 - from, 0) : p.shared_lens ? 1 : 0;
    }
};
__device__ __forceinline__ int length_of(const Params& p, int b) { return p.seq_lens ? min(max(__ldcg(p.seq_lens + b), 0), p.s_max) : p.seq_len; }
__device__ __forceinline__ int shared_of(const Params& p, int b) { return p.shared_lens ? __ldcg(p.shared_lens + b) : 0; }

// equal pieces of a line, the first `r` of them one unit longer
struct Pieces {
    long long q, r;
    __device__ __forceinline__ Pieces(long long total, int pieces) : q(total / pieces), r(total - total / pieces * pieces) {}
    __device__ __forceinline__ long long begin(int i) const { return i * q + min((long long)i, r); }
    __device__ __forceinline__ int piece_of(long long u) const { return (int)(u < r * (q + 1) ? u / (q + 1) : r + (u - r * (q + 1)) / q); }
};

// what the producer says of a chunk
struct Info {
    int key0, len, lo, head;       // its first key, and what is seen
    int flags, pair, slot, parts;  // slot, parts, first_slot: of a piece of a pair that is cut
    int first_slot, pad[3];
};
enum : int { FIRST = 1, LAST = 2, WHOLE = 4 };
enum : int { NO_PAIR = -1, NO_MORE = -2 };   // of a buffer: not for the finisher; nor is any further one

// four columns of O, and with the first of them the LSE
template <int D>
__device__ __forceinline__ void store_row(const Params& p, size_t row, int col, const State& s, float vds) {
    if (p.shared_lens) {
        *reinterpret_cast<float4*>(p.own_o + row * D + col) = s.o;
        if (col == 0) *reinterpret_cast<float2*>(p.own_ml + 2 * row) = make_float2(s.m, s.l);
        return;
    }
    store_output<D>(p.o, p.lse, row, col, s, vds);
}

__device__ __forceinline__ void lds128(uint32_t* r, uint32_t at) {
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void lds64(uint32_t* r, uint32_t at) { asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(at) : "memory"); }
__device__ __forceinline__ void sts128(uint32_t at, int a, int b, int c, int d) { asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory"); }
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

template <int D, int NQ>
__global__ void __launch_bounds__(THREADS, Cfg<D, NQ>::CTAS)
fa_decode_stream_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const Params p) {
    using C = Cfg<D, NQ>;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    const uint32_t base = smem_u32(smem), full = base + C::OFF_BAR, empty = full + 8 * C::STAGES, handed = empty + 8 * C::STAGES, done = handed + 8 * C::BUFFERS,
                   met = done + 8 * C::BUFFERS;
    volatile uint32_t* abort_flag = reinterpret_cast<uint32_t*>(smem + C::OFF_FLAG);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __shared__ uint32_t s_last;
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; s++) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, CONSUMERS);
        }
        for (int i = 0; i < C::BUFFERS; i++) {
            mbar_init(handed + 8 * i, CONSUMERS);
            mbar_init(done + 8 * i, 1);
        }
        mbar_init(met, CONSUMERS);
        *abort_flag = 0;
        fence_mbar_init();
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();   // behind the wait: the kernel of a shared prefix reads without waiting for this one

    float (*const s_o)[CONSUMERS][C::ROWS][C::PITCH] = reinterpret_cast<float (*)[CONSUMERS][C::ROWS][C::PITCH]>(smem + C::OFF_O);   // [BUFFERS]
    float2 (*const s_ml)[CONSUMERS][C::ROWS] = reinterpret_cast<float2 (*)[CONSUMERS][C::ROWS]>(smem + C::OFF_ML);
    volatile int* const s_pair = reinterpret_cast<int*>(smem + C::OFF_PAIR);
    // four columns of a row of the warps' states, added up
    auto sum_of = [&](int buf, int row, int col) {
        State x;
#pragma unroll
        for (int w = 0; w < CONSUMERS; w++) {
            const float2 ml = s_ml[buf][w][row];
            x.add(ml.x, ml.y, *reinterpret_cast<const float4*>(&s_o[buf][w][row][col]));
        }
        return x;
    };
    if (warp == FINISHER) {
        // ------------------------------------------------------------------------ whole pairs, while the next ones are attended to
        const float vds = p.sv ? p.v_descale * ld_f32(p.sv) : p.v_descale;
        for (uint32_t nth = 0;; nth++) {
            const int buf = nth % C::BUFFERS;
            if (!mbar_wait_warp(handed + 8 * buf, nth / C::BUFFERS & 1, abort_flag, ST_STREAM_FINISH)) break;
            const int pair = s_pair[buf];
            if (pair == NO_MORE) break;
            if (pair >= 0)
                for (int i = lane; i < p.group * (D / 4); i += 32)
                    store_row<D>(p, (size_t)pair * p.group + i / (D / 4), i % (D / 4) * 4, sum_of(buf, i / (D / 4), i % (D / 4) * 4), vds);
            __syncwarp();
            if (lane == 0) mbar_arrive(done + 8 * buf);
        }
    } else if (warp == PRODUCER) {
        // ------------------------------------------------------------------------------------------------- producer
        const bool leader = lane == 0;
        if (leader) {
            prefetch_tmap(&tmap_k);
            prefetch_tmap(&tmap_v);
        }
        // lengths of sequences lane, lane + 32, ..; larger batches read theirs again
        constexpr int KEPT = 4;
        int lens[KEPT], shared[KEPT];
#pragma unroll
        for (int i = 0; i < KEPT; i++) {
            const int b = 32 * i + lane;
            lens[i] = b < p.batch ? length_of(p, b) : 0;
            shared[i] = b < p.batch ? shared_of(p, b) : 0;
        }
        auto read = [&](int b0, int& len, int& sh) {   // of sequence b0 + lane, b0 a multiple of 32
            if (b0 < 32 * KEPT) {
                len = lens[0];
                sh = shared[0];
#pragma unroll
                for (int i = 1; i < KEPT; i++)
                    if (b0 == 32 * i) { len = lens[i]; sh = shared[i]; }
            } else {
                len = b0 + lane < p.batch ? length_of(p, b0 + lane) : 0;
                sh = b0 + lane < p.batch ? shared_of(p, b0 + lane) : 0;
            }
        };
        long long total = 0;
        for (int b0 = 0; b0 < p.batch; b0 += 32) {
            int len, sh;
            read(b0, len, sh);
            total += __reduce_add_sync(0xffffffffu, b0 + lane < p.batch ? (uint32_t)Span(p, len, sh).n : 0u);   // 32 of at most 2^25
        }
        total *= p.hkv;
        const Pieces cut(total, gridDim.x);
        long long u = cut.begin(blockIdx.x);
        const long long end = cut.begin(blockIdx.x + 1);
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        while (u < end && ok) {
            // the pair that unit u falls in: the sequence, its length and what lies before it come from one reading
            int b = -1, len = 0, sh = 0;
            long long seq_u0 = 0;
            for (int b0 = 0; b0 < p.batch; b0 += 32) {
                int len_l, sh_l;
                read(b0, len_l, sh_l);
                const uint32_t n = b0 + lane < p.batch ? (uint32_t)Span(p, len_l, sh_l).n : 0u;
                uint32_t incl = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += y;
                }
                const uint32_t past = __ballot_sync(0xffffffffu, seq_u0 + (long long)incl * p.hkv > u);
                if (past) {
                    const int at = __ffs(past) - 1;
                    seq_u0 += (long long)__shfl_sync(0xffffffffu, incl - n, at) * p.hkv;
                    b = b0 + at;
                    len = __shfl_sync(0xffffffffu, len_l, at);
                    sh = __shfl_sync(0xffffffffu, sh_l, at);
                    break;
                }
                seq_u0 += (long long)__shfl_sync(0xffffffffu, incl, 31) * p.hkv;
            }
            if (b < 0) break;   // lengths that have changed meanwhile
            const Span x(p, len, sh);
            for (int kvh = (int)((u - seq_u0) / x.n); kvh < p.hkv && u < end && ok; kvh++) {
                const long long pair_u0 = seq_u0 + (long long)kvh * x.n;
                const int c_begin = (int)(u - pair_u0), c_end = (int)min((long long)x.n, c_begin + (end - u));
                const bool whole = c_begin == 0 && c_end == x.n;
                int parts = 1, first = 0;
                if (!whole) {
                    first = cut.piece_of(pair_u0);
                    parts = cut.piece_of(pair_u0 + x.n - 1) - first + 1;
                }
                const int pair = b * p.hkv + kvh, slot = 2 * blockIdx.x + (c_begin == 0 ? 1 : 0);
                int entry = 0, entries_from = -32 * CHUNK;   // lane i: the table's entry for chunk entries_from + i
                for (int c = c_begin; c < c_end; c++) {
                    if (p.block_table && (c - entries_from >= 32 || c == c_begin)) {
                        entries_from = c;
                        const int ci = c + lane, key = (ci < x.head_chunks ? ci : ci + x.skip) * CHUNK;
                        entry = -1;
                        if (ci < c_end && key < x.len) {
                            const int page = __ldcg(p.block_table + (size_t)b * p.max_pages + p.page.div((uint32_t)key));
                            if (page >= 0 && page < p.num_pages) entry = page;
                        }
                    }
                    const int key0 = (c < x.head_chunks ? c : c + x.skip) * CHUNK;
                    int row = key0, z = b * p.hkv + kvh;
                    if (p.block_table) {
                        const int page = __shfl_sync(0xffffffffu, entry, c - entries_from);
                        row = key0 - (int)p.page.div((uint32_t)key0) * p.page_size;
                        z = page < 0 ? -1 : page * p.hkv + kvh;   // -1: outside the map, which arrives as zeros
                    }
                    ok = mbar_wait_warp(empty + 8 * s, ph ^ 1, abort_flag, ST_STREAM_LOAD);
                    if (!ok) break;
                    if (leader) {
                        const uint32_t at = base + C::OFF_INFO + 48 * s, bar = full + 8 * s;
                        const int flags = (c == c_begin ? FIRST : 0) | (c == c_end - 1 ? LAST : 0) | (whole ? WHOLE : 0);
                        sts128(at, key0, x.len, x.lo, x.head);
                        sts128(at + 16, flags, pair, slot, parts);
                        sts128(at + 32, 2 * first + 1, 0, 0, 0);
                        const uint32_t q_bytes = c == c_begin ? (uint32_t)p.group * D : 0u;
                        mbar_arrive_expect_tx(bar, 2 * C::TILE + q_bytes);
                        tma_load_3d(base + s * C::TILE, &tmap_k, bar, 0, row, z);
                        tma_load_3d(base + C::OFF_V + s * C::TILE, &tmap_v, bar, 0, row, z);
                        if (q_bytes) bulk_load(base + C::OFF_Q + s * C::ROWS * D, p.q + (size_t)pair * q_bytes, q_bytes, bar);
                    }
                    __syncwarp();
                    if (++s == C::STAGES) { s = 0; ph ^= 1; }
                }
                u += c_end - c_begin;
            }
        }
        // a chunk of no pair says that there is no more
        if (ok && mbar_wait_warp(empty + 8 * s, ph ^ 1, abort_flag, ST_STREAM_LOAD) && leader) {
            sts128(base + C::OFF_INFO + 48 * s + 16, 0, -1, 0, 0);
            mbar_arrive(full + 8 * s);
        }
    } else {
        // ------------------------------------------------------------------------------------------------ consumers
        const int g = lane >> 2, t = lane & 3;   // fragment coordinates
        if (!p.shared_lens) {   // a sequence without keys is on nobody's piece
            for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
                if (length_of(p, b) > 0) continue;
                const int rows = p.hkv * p.group;
                for (int i = threadIdx.x; i < rows * D; i += 32 * CONSUMERS) p.o[(size_t)b * rows * D + i] = __float2half_rn(0.f);
                if (p.lse)
                    for (int i = threadIdx.x; i < rows; i += 32 * CONSUMERS) p.lse[(size_t)b * rows + i] = -INFINITY;
            }
        }
        float scale_log2 = p.scale_log2;
        if (p.sq) scale_log2 *= ld_f32(p.sq);
        if (p.sk) scale_log2 *= ld_f32(p.sk);
        const float vds = p.sv ? p.v_descale * ld_f32(p.sv) : p.v_descale;
        // this lane's bytes of a row in its chunk: rows g and g + 8 of K, 2t, 2t + 1, 2t + 8 and 2t + 9 of V of the warp's 16, at the swizzle's places
        const int k_row = 16 * warp + g, v_row = 16 * warp + 2 * t;
        auto k_at = [&](int row, int h) -> uint32_t { return row * D + (D == 128 ? ((2 * t + h) ^ (row & 7)) << 4 : (t ^ ((row >> 1) & 3)) << 4); };
        auto v_at = [&](int row) -> uint32_t { return row * D + (D == 128 ? (g ^ (row & 7)) << 4 : (((g >> 1) ^ ((row >> 1) & 3)) << 4) + 8 * (g & 1)); };
        uint32_t qf[NQ][C::KW];
        float m[NQ][2], l[NQ][2], acc[NQ][C::MT][4];
        int s = 0;
        uint32_t ph = 0;
        // all consumers: a bounded wait, so that a warp that gives up strands nobody
        uint32_t met_ph = 0, nth = 0;   // nth: pairs and pieces that have ended
        auto meet = [&]() -> bool {
            __syncwarp();
            if (lane == 0) mbar_arrive(met);
            const bool ok = mbar_wait_warp(met, met_ph, abort_flag, ST_STREAM_MEET);
            met_ph ^= 1;
            return ok;
        };
        for (;;) {
            if (!mbar_wait_warp(full + 8 * s, ph, abort_flag, ST_STREAM_USE)) break;
            const Info& info = *reinterpret_cast<const Info*>(smem + C::OFF_INFO + 48 * s);
            const int4 seen = *reinterpret_cast<const int4*>(&info.key0), what = *reinterpret_cast<const int4*>(&info.flags);
            const int flags = what.x, pair = what.y, slot = what.z, parts = what.w, first_slot = info.first_slot;
            if (pair < 0) break;
            if (flags & FIRST) {
                const uint32_t qb = base + C::OFF_Q + s * C::ROWS * D + (D / 4) * t;
#pragma unroll
                for (int n = 0; n < NQ; n++) {
#pragma unroll
                    for (int w = 0; w < C::KW; w += 4) lds128(qf[n] + w, qb + (8 * n + g) * D + 4 * w);
                    if (8 * n + g >= p.group)
#pragma unroll
                        for (int w = 0; w < C::KW; w++) qf[n][w] = 0u;
#pragma unroll
                    for (int e = 0; e < 2; e++) { m[n][e] = -INFINITY; l[n][e] = 0.f; }
#pragma unroll
                    for (int j = 0; j < C::MT; j++) acc[n][j][0] = acc[n][j][1] = acc[n][j][2] = acc[n][j][3] = 0.f;
                }
            }
            const int key0 = seen.x + 16 * warp;   // this warp's keys
            const bool cut = key0 + 16 > seen.y || (key0 < seen.z && key0 + 16 > seen.w);
            const bool none = key0 >= seen.y || (key0 >= seen.w && key0 + 16 <= seen.z);
            auto sees = [&](int key) { return key < seen.y && (key >= seen.z || key < seen.w); };
            uint32_t vr[4][C::VW];
            float sc[NQ][4];
            if (!none) {
                uint32_t kr[2][C::KW];
                const uint32_t kb = base + s * C::TILE, vb = base + C::OFF_V + s * C::TILE;
#pragma unroll
                for (int r = 0; r < 2; r++)
#pragma unroll
                    for (int h = 0; h < D / 64; h++) lds128(kr[r] + 4 * h, kb + k_at(k_row + 8 * r, h));
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int row = v_row + (r & 1) + 8 * (r >> 1);
                    if (D == 128) lds128(vr[r], vb + v_at(row));
                    else lds64(vr[r], vb + v_at(row));
                }
                // one accumulator per k-step: independent MMAs instead of a chain
#pragma unroll
                for (int n = 0; n < NQ; n++) {
                    float part[D / 32][4];
#pragma unroll
                    for (int ks = 0; ks < D / 32; ks++)
                        mma_e4m3_zero(part[ks], kr[0][2 * ks], kr[1][2 * ks], kr[0][2 * ks + 1], kr[1][2 * ks + 1], qf[n][2 * ks], qf[n][2 * ks + 1]);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float x = part[0][e];
#pragma unroll
                        for (int ks = 1; ks < D / 32; ks++) x += part[ks][e];
                        sc[n][e] = x * scale_log2;
                    }
                }
            }
            // all that the stage holds is in registers
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + 8 * s);
            if (++s == C::STAGES) { s = 0; ph ^= 1; }
            if (!none) {
                if (cut) {   // keys that are not seen may hold anything: their values must not meet a weight of zero
#pragma unroll
                    for (int n = 0; n < NQ; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (!sees(key0 + g + 8 * (e >> 1))) sc[n][e] = -INFINITY;
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (!sees(key0 + 2 * t + (r & 1) + 8 * (r >> 1)))
#pragma unroll
                            for (int w = 0; w < C::VW; w++) vr[r][w] = 0u;
                }
                // sc[n][e]: key g (e < 2) or g + 8, query 8n + 2t + (e & 1)
                float mx[NQ][2];
                bool bump = false;
#pragma unroll
                for (int n = 0; n < NQ; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        mx[n][e] = fmaxf(sc[n][e], sc[n][e + 2]);
                        bump = bump || mx[n][e] > m[n][e] + LAG;
                    }
                if (__any_sync(0xffffffffu, bump)) {   // rare once a few chunks are in
#pragma unroll
                    for (int n = 0; n < NQ; n++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) mx[n][e] = fmaxf(mx[n][e], __shfl_xor_sync(0xffffffffu, mx[n][e], o));
                            const float m_new = fmaxf(m[n][e], mx[n][e]);
                            const float f = m[n][e] == -INFINITY ? 0.f : exp2_fast(m[n][e] - m_new);
                            m[n][e] = m_new;
                            l[n][e] *= f;
#pragma unroll
                            for (int j = 0; j < C::MT; j++) {
                                acc[n][j][e] *= f;
                                acc[n][j][e + 2] *= f;
                            }
                        }
                }
                uint32_t pf[NQ][2];   // P^T: rows (keys) 2t, 2t + 1 and 2t + 8, 2t + 9 of column g
#pragma unroll
                for (int n = 0; n < NQ; n++) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        w[e] = sc[n][e] == -INFINITY ? 0.f : exp2_fast(sc[n][e] - m[n][e & 1]);
                        l[n][e & 1] += w[e];
                    }
                    pf[n][0] = transpose_8x8(half2_bits(w[0], w[1]));
                    pf[n][1] = transpose_8x8(half2_bits(w[2], w[3]));
                }
                // rows g and g + 8 of tile j of O^T are d = (D/8) g + 2j and + 1
#pragma unroll
                for (int w = 0; w < C::VW; w++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t sel = h ? 0x7362 : 0x5140;   // bytes (2h, 2h + 1) of two keys, interleaved
                        uint32_t a[4];
                        e4m3_to_half(__byte_perm(vr[0][w], vr[1][w], sel), a[0], a[1]);
                        e4m3_to_half(__byte_perm(vr[2][w], vr[3][w], sel), a[2], a[3]);
#pragma unroll
                        for (int n = 0; n < NQ; n++) mma_f16(acc[n][2 * w + h], a, pf[n][0], pf[n][1]);
                    }
            }
            if (!(flags & LAST)) continue;

            // ---- the four warps' states of the pair
            const int sum = nth % C::BUFFERS;
            if (!mbar_wait_warp(done + 8 * sum, (nth / C::BUFFERS & 1) ^ 1, abort_flag, ST_STREAM_USE)) break;
            nth++;
#pragma unroll
            for (int n = 0; n < NQ; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], o);
                    const int row = 8 * n + 2 * t + e;
                    if (g == 0) s_ml[sum][warp][row] = make_float2(m[n][e], l[n][e]);
                    if (row < p.group) {
#pragma unroll
                        for (int j = 0; j < C::MT; j++)
                            *reinterpret_cast<float2*>(&s_o[sum][warp][row][(D / 8) * g + 2 * j]) = make_float2(acc[n][j][e], acc[n][j][e + 2]);
                    }
                }
            if (threadIdx.x == 0) s_pair[sum] = flags & WHOLE ? pair : NO_PAIR;
            if (!(flags & WHOLE)) {   // a piece: the consumers themselves, for the last one of a pair has many to add up
                if (!meet()) break;
                for (int i = threadIdx.x; i < p.group * (D / 4); i += 32 * CONSUMERS) {
                    const int row = i / (D / 4), col = i % (D / 4) * 4;
                    const State x = sum_of(sum, row, col);
                    const size_t at = (size_t)slot * C::ROWS + row;
                    __stcg(reinterpret_cast<float4*>(p.ws_o + at * D + col), x.o);
                    if (col == 0) __stcg(reinterpret_cast<float2*>(p.ws_ml + at * 2), make_float2(x.m, x.l));
                }
                __threadfence();
                if (!meet()) break;
                if (threadIdx.x == 0) {
                    s_last = atomicAdd(p.arrivals + pair, 1u) == (uint32_t)(parts - 1);
                    if (s_last) p.arrivals[pair] = 0;   // for the next launch
                }
                if (!meet()) break;
                if (s_last) {
                    __threadfence();
                    for (int i = threadIdx.x; i < p.group * (D / 4); i += 32 * CONSUMERS) {
                        const int row = i / (D / 4), col = i % (D / 4) * 4;
                        State x;   // slots: first_slot, then the even ones of the CTAs behind
                        x.add_all<D>(p.ws_ml, p.ws_o, parts, col, [&](int k) { return (size_t)(k == 0 ? first_slot : first_slot + 2 * k - 1) * C::ROWS + row; });
                        store_row<D>(p, (size_t)pair * p.group + row, col, x, vds);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(handed + 8 * sum);
        }
        // (having given up, a consumer finds the others and the finisher giving up as well)
        const int sum = nth % C::BUFFERS;
        if (mbar_wait_warp(done + 8 * sum, (nth / C::BUFFERS & 1) ^ 1, abort_flag, ST_STREAM_USE)) {
            if (threadIdx.x == 0) s_pair[sum] = NO_MORE;
            __syncwarp();
            if (lane == 0) mbar_arrive(handed + 8 * sum);
        }
    }
    __syncthreads();
    const uint32_t code = *abort_flag;
    if (code != 0) {
        if (threadIdx.x == 0) atomicCAS(p.status, 0u, code);
        for (int i = 0; i < 200; i++) __nanosleep(1000);   // let copies already in flight land
    }
}

// chunks that a pair can have at most
long long most_chunks(const StreamArgs& a) {
    const long long all = ((long long)(a.seq_lens ? a.s_max : a.seq_len) + CHUNK - 1) / CHUNK;
    if (a.shared_lens) return all > 0 ? all : 1;
    const long long seen = a.window > 0 ? ((long long)a.sinks + CHUNK - 1) / CHUNK + ((long long)a.window + CHUNK - 1) / CHUNK + 1 : all;
    return seen < all ? seen : all;
}
int rows_of(const StreamArgs& a) { return a.q_heads / a.kv_heads <= 8 ? 8 : 16; }
int grid_of(const StreamArgs& a) {
    const long long units = most_chunks(a) * a.batch * a.kv_heads, resident = (long long)sms_of_current_device() * Cfg<128, 1>::CTAS;
    return (int)(units < 1 ? 1 : units < resident ? units : resident);
}

template <int D, int NQ>
cudaError_t run(const StreamArgs& a, const Params& p, const CUtensorMap& k, const CUtensorMap& v) {
    using C = Cfg<D, NQ>;
    const cudaError_t e = cudaFuncSetAttribute(fa_decode_stream_kernel<D, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    return launch_pdl(fa_decode_stream_kernel<D, NQ>, dim3((unsigned)grid_of(a)), dim3(THREADS), C::SMEM, a.stream, k, v, p);
}

}  // namespace

int sms_of_current_device() {
    static std::atomic<int> known[64];
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return sms;
    if (const int n = known[dev].load(std::memory_order_relaxed)) return n;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) known[dev].store(sms, std::memory_order_relaxed);
    return sms;
}

size_t stream_workspace_bytes(const StreamArgs& a) { return (size_t)grid_of(a) * 2 * rows_of(a) * (a.hd + 2) * sizeof(float); }
size_t stream_arrivals(const StreamArgs& a) { return (size_t)a.batch * a.kv_heads; }

cudaError_t launch_stream(const StreamArgs& a) {
    Params p;
    p.q = static_cast<const uint8_t*>(a.q);
    p.o = static_cast<__half*>(a.o);
    p.lse = a.lse;
    p.seq_lens = a.seq_lens;
    p.shared_lens = a.shared_lens;
    p.batch = a.batch; p.hkv = a.kv_heads; p.group = a.q_heads / a.kv_heads;
    p.s_max = a.s_max; p.seq_len = a.seq_len; p.window = a.window; p.sinks = a.sinks;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.v_descale = a.v_descale;
    p.sq = a.scale_q_dev; p.sk = a.scale_k_dev; p.sv = a.scale_v_dev;
    p.block_table = a.block_table;
    p.max_pages = a.max_pages; p.num_pages = a.num_pages; p.page_size = a.page_size;
    p.page = FastDiv(a.block_table ? (uint32_t)a.page_size : 1u);
    p.ws_ml = static_cast<float*>(a.workspace);
    p.ws_o = p.ws_ml + (size_t)grid_of(a) * 2 * rows_of(a) * 2;
    p.arrivals = a.arrivals;
    p.own_o = a.own_o; p.own_ml = a.own_ml;
    p.status = status_word();
    if (!p.status) return cudaErrorInvalidSymbol;
    const uint64_t outer = (uint64_t)(a.block_table ? a.num_pages : a.batch) * a.kv_heads, rows = (uint64_t)(a.block_table ? a.page_size : a.s_max);
    const CUtensorMapSwizzle swizzle = a.hd == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    CUtensorMap k, v;
    if (!make_tmap_u8_3d(&k, a.k_cache, outer, rows, a.hd, CHUNK, a.hd, swizzle) || !make_tmap_u8_3d(&v, a.v_cache, outer, rows, a.hd, CHUNK, a.hd, swizzle)) return cudaErrorInvalidValue;
    const bool two = rows_of(a) == 16;
    if (a.hd == 64) return two ? run<64, 2>(a, p, k, v) : run<64, 1>(a, p, k, v);
    return two ? run<128, 2>(a, p, k, v) : run<128, 1>(a, p, k, v);
}

namespace {
cudaError_t launch_with(const void* args, const CallScratch& scratch) {
    StreamArgs a = *static_cast<const StreamArgs*>(args);
    a.workspace = scratch.workspace;
    a.arrivals = scratch.zeros;
    return launch_stream(a);
}
}  // namespace

StreamArgs stream_args(const fa_decode_args_t& g, int s_max) {
    StreamArgs a = {};
    a.q = g.q; a.k_cache = g.k_cache; a.v_cache = g.v_cache; a.o = g.o; a.lse = static_cast<float*>(g.l_out);
    a.seq_lens = g.seq_lens;
    a.batch = g.batch; a.q_heads = g.q_heads; a.kv_heads = g.kv_heads; a.hd = g.head_dim; a.s_max = s_max; a.seq_len = g.seq_len;
    a.scale = g.scale;
    a.v_descale = g.v_descale == 0.0f ? 1.0f : g.v_descale;
    a.scale_q_dev = g.scale_q_dev; a.scale_k_dev = g.scale_k_dev; a.scale_v_dev = g.scale_v_dev;
    a.block_table = g.block_table; a.page_size = g.page_size; a.max_pages = g.max_pages_per_seq; a.num_pages = g.num_pages;
    a.stream = reinterpret_cast<cudaStream_t>(g.stream);
    return a;
}

fa_status_t check_stream(fa_ctx_t* ctx, const char* who, const fa_decode_args_t* g, int& s_max) {
    const fa_status_t ok = check_decode(ctx, who, g, 16, s_max);
    if (ok != FA_OK) return ok;
    if ((long long)(g->block_table ? g->num_pages : g->batch) * g->kv_heads > 0x7fffffffLL)
        return refuse(ctx, who, FA_ERR_UNSUPPORTED_SHAPE, "kv_heads times the pages of a pool (or sequences of a contiguous cache) must be below 2^31");
    if ((long long)g->batch * g->q_heads > 0x7fffffffLL) return refuse(ctx, who, FA_ERR_UNSUPPORTED_SHAPE, "batch times q_heads must be below 2^31");
    for (const void* p : {(const void*)g->l_out, (const void*)g->seq_lens, (const void*)g->block_table, (const void*)g->scale_q_dev, (const void*)g->scale_k_dev, (const void*)g->scale_v_dev})
        if (reinterpret_cast<uintptr_t>(p) & 3) return refuse(ctx, who, FA_ERR_INVALID_ARG, "l_out, seq_lens, block_table and scales must be 4-byte aligned");
    return FA_OK;
}

fa_status_t launch_stream_call(fa_ctx_t* ctx, const char* who, const StreamArgs& a) {
    return call_with_scratch(ctx, who, a.stream, stream_workspace_bytes(a), stream_arrivals(a), launch_with, &a);
}

}  // namespace fa_sm100

extern "C" fa_status_t fa_decode_window(fa_ctx_t* ctx, const fa_decode_args_t* g, int window, int sinks) {
    const char* who = "fa_decode_window";
    if (!ctx) return FA_ERR_INVALID_ARG;
    int s_max = 0;
    const fa_status_t ok = fa_sm100::check_stream(ctx, who, g, s_max);
    if (ok != FA_OK) return ok;
    if (window < 0 || sinks < 0) return fa_sm100::refuse(ctx, who, FA_ERR_INVALID_ARG, "window and sinks must be >= 0");
    fa_sm100::StreamArgs a = fa_sm100::stream_args(*g, s_max);
    a.window = window;
    a.sinks = sinks;
    return fa_sm100::launch_stream_call(ctx, who, a);
}
