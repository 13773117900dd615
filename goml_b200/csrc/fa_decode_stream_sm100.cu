// fa_decode_stream_sm100.cu — FP8 decode attention over a part of each sequence's keys (sm_100a): a window with the first tokens (fa_decode_window), or what a
// sequence has behind a shared prefix (the first kernel of fa_decode_shared).
//
// For one query the keys that it sees are two runs, [0, head) and [lo, len); the units of 32 (head dim 64: 64) keys that hold any of them, sinks first, are the sequence's line, and the
// lines of all pairs (sequence, kv head) one behind another are cut into equal pieces, one for every resident CTA.  Each byte is used once, 4 flops of the tensor cores
// for each query head that shares it: bound by memory.  So
//  * one warp of a CTA (the producer) walks the piece and hands units to two others, two of them to each ahead, with one tensor-map copy for K and V (swizzled, so that fragments are
//    read without bank conflicts; rows past a cache's end and pages that the pool does not have arrive as zeros), across the ends of pairs.  What belongs to a unit, masks and ends of
//    pairs among it, it writes beside it, so that
//  * a warp takes units whole and looks at nothing else: S^T = K Q^T (m16n8k32 on the codes), a running maximum that may lag by 2^6 (its rescaling is rare), P in fp16,
//    O^T += V^T P^T (m16n8k16 on V converted in registers).  A pair of few units is one warp's, which writes its O; the units of a longer one go round all.
//  * The states of such a pair meet in shared memory, where one more warp adds them up while the next pair is attended to.  Pieces of a pair that is cut meet in a workspace, where the
//    CTA that is last adds them up in order: results do not depend on timing.
// Few keys or few sequences are slower than in fa_decode, whose parts of a pair meet in a cluster's shared memory instead of L2: window 0, 32 query heads, us in CUDA graphs, fa_decode / here: one sequence of 1000 keys,
// 8 kv heads, 8.3 / 12.1, 32 kv heads 6.8 / 13.7; many keys are not: 128 of 4000, 8 kv heads, 169.5 / 165.9, 32 of 4000, 32 kv heads, 201 / 165; one of 16000, one kv head with 16 query heads, 72.5 / 27.8.
// Measured: 128 sequences that see 4100 of 6000 to 8000 keys, 32 query and 8 kv heads of 128, in pages: 168 us, 6.3 TB/s, 0.96 of the copy rate (four warps of a CTA on one unit of 64 keys 174 to
// 199).  One sequence of 1028, 32 heads: 11 us, which are the launch, the lengths' chain, a first load and the sums.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>
#include <initializer_list>

#include "../../include/fa_sm120.h"
#include "fa_decode_mma.cuh"
#include "fa_decode_stream.h"
#include "fa_line_pieces.h"
#include "fa_scratch_call.h"
#include "pdl.cuh"
#include "row_items.cuh"
#include "sm100_ptx.cuh"
#include "tmap.cuh"

namespace fa_sm100 {

namespace {

using namespace sm100;

constexpr int CONSUMERS = 2, PRODUCER = CONSUMERS, THREADS = 32 * (CONSUMERS + 2);
constexpr int DEPTH = 2;      // units of a consumer that are loaded or on their way
constexpr int RECORDS = 4;    // pairs that end, on their way to the finisher
// Units of a pair up to which they are one warp's.  Of 2, 4 and 8: 300 sequences of 200 keys, 8 kv heads, 35.8 us, 37.2, 38.6; 256 of 500 of 64 34.4, 34.1, 38.9; 1000 of 128 62.8, 63.7, 64.8.
constexpr int ALONE = 2;
constexpr float LAG = 6.0f;   // log2 units
// Pieces of a pair, on average.  Of 8, 16, 32 and 64: one sequence of 8000 keys, 8 kv heads, 20.9 us, 16.0, 16.0, 17.5; of 30000 49.6, 30.6, 24.6, 21.8; one of 1028, 32 heads, 12.5, 12.2, 12.2,
// 12.2; two of 1500, one kv head, 16.5, 15.1, 17.5, 16.2.
constexpr int MAX_PARTS = 32;
enum : uint32_t { ST_STREAM_LOAD = 0x241, ST_STREAM_USE = 0x242, ST_STREAM_FINISH = 0x243, ST_STREAM_SMEM = 0x244 };

template <int D, int NQ>
struct Cfg {
    static constexpr int TILES = D == 128 ? 2 : 4;     // of 16 keys in a unit
    static constexpr int UNIT = 16 * TILES;            // keys (page sizes are multiples of it)
    static constexpr int ROWS = 8 * NQ;                // query columns
    static constexpr int PITCH = NQ == 1 ? D + 4 : D;  // floats of a row of a warp's state (of 16 rows, all that fits)
    static constexpr int BYTES = UNIT * D;             // of a unit of K or V
    static constexpr int KW = D / 16;                  // words of a lane's share of a K row
    static constexpr int MT = D / 16;                  // 16-row tiles of O^T
    static constexpr int VW = D / 32;                  // words of a lane's share of a V row
    static constexpr int STAGES = CONSUMERS * DEPTH;
    static constexpr int OFF_V = STAGES * BYTES;
    static constexpr int OFF_Q = 2 * STAGES * BYTES;
    static constexpr int OFF_INFO = OFF_Q + STAGES * ROWS * D;
    static constexpr int OFF_RECORD = OFF_INFO + STAGES * 32;
    static constexpr int OFF_BAR = OFF_RECORD + RECORDS * 32;
    static constexpr int BARRIERS = 2 * STAGES + CONSUMERS + 2 * RECORDS;
    static constexpr int OFF_FLAG = OFF_BAR + 8 * BARRIERS;
    static constexpr int OFF_START = OFF_FLAG + 8;     // where the piece starts, and the sums that find it
    static constexpr int OFF_LEFT = (OFF_START + 32 + 8 * (THREADS / 32) + 15) & -16;   // what is left to do when all roles have ended: two records and a word
    static constexpr int OFF_O = (OFF_LEFT + 80 + 127) & -128;
    static constexpr int OFF_ML = OFF_O + CONSUMERS * ROWS * PITCH * 4;
    static constexpr int SMEM = OFF_ML + CONSUMERS * ROWS * 8;
    static constexpr int CTAS = NQ == 1 ? 4 : 3;       // resident on an SM
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

// The keys that a sequence sees, as units: `head` keys in the first `head_units`, then those from unit head_units + skip on.
template <int UNIT>
struct Span {
    int len, lo, head, head_units, skip, n;
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
        // (of nothing behind the prefix, the unit of the last key: every pair has one, and with it a state)
        const int first = max(min(lo, len - 1), 0) / UNIT;
        head_units = (head + UNIT - 1) / UNIT;
        const int from = max(first, head_units);
        skip = from - head_units;
        n = len > 0 ? head_units + max((len - 1) / UNIT + 1 - from, 0) : p.shared_lens ? 1 : 0;
    }
};
__device__ __forceinline__ int length_of(const Params& p, int b) { return p.seq_lens ? min(max(__ldcg(p.seq_lens + b), 0), p.s_max) : p.seq_len; }
__device__ __forceinline__ int shared_of(const Params& p, int b) { return p.shared_lens ? __ldcg(p.shared_lens + b) : 0; }

// what the producer says of a unit
struct Info {
    int key0, len, lo, head;   // its first key, and what is seen
    int flags, pair, record, pad;
};
enum : int { FIRST = 1, LAST = 2, DIRECT = 4 };   // of the pair to this warp; its whole
// and of a pair that ends in shared memory: the warps that have states of it (`count` of them, from `first_warp` round), and of a piece its slot, the number of pieces and the first one's slot
struct Record {
    int pair, first_warp, count, kind;
    int slot, parts, first_slot, pad;
};
enum : int { WHOLE = 0, PIECE = 1, TAIL = 2 };   // TAIL: a piece that is the last of its CTA
enum : int { NO_MORE = -1 };   // pair of a unit or a record

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

__device__ __forceinline__ void mbar_arrive_count(uint32_t bar, uint32_t n) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(bar), "r"(n) : "memory");
}

template <int D, int NQ>
__global__ void __launch_bounds__(THREADS, Cfg<D, NQ>::CTAS)
fa_decode_stream_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const Params p) {
    using C = Cfg<D, NQ>;
    using Span = Span<C::UNIT>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_u32(smem);
    const uint32_t full = base + C::OFF_BAR;                  // [CONSUMERS][DEPTH] a unit has landed
    const uint32_t empty = full + 8 * C::STAGES;              // [CONSUMERS][DEPTH] ... and is used
    const uint32_t freed = empty + 8 * C::STAGES;             // [CONSUMERS] a warp's state is added up
    const uint32_t handed = freed + 8 * CONSUMERS;            // [RECORDS] the states of a record are there
    const uint32_t taken = handed + 8 * RECORDS;              // [RECORDS] ... and are added up
    volatile uint32_t* abort_flag = reinterpret_cast<uint32_t*>(smem + C::OFF_FLAG);
    // [0]: a piece whose pair is to be added up; [1]: a tail whose states lie in shared memory.  parts 0: there is none
    Record* const left = reinterpret_cast<Record*>(smem + C::OFF_LEFT);
    volatile int* const s_last = reinterpret_cast<int*>(smem + C::OFF_LEFT + 64);
    float (*const s_o)[C::PITCH] = reinterpret_cast<float (*)[C::PITCH]>(smem + C::OFF_O);   // the warps' rows
    float2* const s_ml = reinterpret_cast<float2*>(smem + C::OFF_ML);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; s++) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int w = 0; w < CONSUMERS; w++) mbar_init(freed + 8 * w, 1);
        for (int i = 0; i < RECORDS; i++) {
            mbar_init(handed + 8 * i, CONSUMERS + 1);   // the producer arrives for itself and for warps without a state
            mbar_init(taken + 8 * i, 1);
        }
        *abort_flag = base & 1023u ? ST_STREAM_SMEM : 0;
        fence_mbar_init();
        prefetch_tmap(&tmap_k);
        prefetch_tmap(&tmap_v);
        left[0].parts = left[1].parts = 0;
    }
    pdl_wait();
    pdl_trigger();   // behind the wait: the kernel of a shared prefix reads without waiting for this one

    // ---- where this CTA's piece starts: every thread adds up the units of a run of sequences
    struct Start {
        long long before;         // units in front of the sequence that the piece starts in
        int b, len, shared, pad;
    };
    Start* const s_start = reinterpret_cast<Start*>(smem + C::OFF_START);
    long long* const s_sums = reinterpret_cast<long long*>(smem + C::OFF_START + 32);
    long long total = 0, u, end;
    Pieces cut(0, 1);
    {
        const int run = (p.batch + THREADS - 1) / THREADS, b0 = min((int)threadIdx.x * run, p.batch), b1 = min(b0 + run, p.batch);
        long long mine = 0;
#pragma unroll 4
        for (int b = b0; b < b1; b++) mine += Span(p, length_of(p, b), shared_of(p, b)).n;
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        if (lane == 31) s_sums[warp] = upto;
        if (threadIdx.x == 0) s_start->b = p.batch;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 32; w++) {
            if (w < warp) upto += s_sums[w];
            total += s_sums[w];
        }
        cut = Pieces(total * p.hkv, gridDim.x);
        u = cut.begin(blockIdx.x);
        end = cut.begin(blockIdx.x + 1);
        if (mine && u < end && (upto - mine) * p.hkv <= u && u < upto * p.hkv) {
            long long before = upto - mine;
            for (int b = b0; b < b1; b++) {
                const int len = length_of(p, b), shared = shared_of(p, b), n = Span(p, len, shared).n;
                if (u < (before + n) * p.hkv) {
                    *s_start = Start{before * p.hkv, b, len, shared, 0};
                    break;
                }
                before += n;
            }
        }
        __syncthreads();
    }

    // item i (a row, four columns) of the warps' states of a record: O of a whole pair, or a state in the workspace
    auto add_states = [&](const Record& r, int i, float vds) {
        const int row = i / (D / 4), col = i % (D / 4) * 4;
        State x;
        for (int k = 0, w = r.first_warp; k < r.count; k++, w = w + 1 < CONSUMERS ? w + 1 : 0) {
            const float2 ml = s_ml[w * C::ROWS + row];
            x.add(ml.x, ml.y, *reinterpret_cast<const float4*>(&s_o[w * C::ROWS + row][col]));
        }
        if (r.kind == WHOLE) {
            store_row<D>(p, (size_t)r.pair * p.group + row, col, x, vds);
        } else {
            const size_t at = (size_t)r.slot * C::ROWS + row;
            __stcg(reinterpret_cast<float4*>(p.ws_o + at * D + col), x.o);
            if (col == 0) __stcg(reinterpret_cast<float2*>(p.ws_ml + at * 2), make_float2(x.m, x.l));
        }
    };
    // Whether the piece is the last of its pair to be done, by one thread behind a barrier with those that have written its state: one addition that releases what they have
    // written and acquires what the others have.
    auto last_of = [&](const Record& r) -> bool {
        uint32_t before;
        asm volatile("atom.global.acq_rel.gpu.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(p.arrivals + r.pair) : "memory");
        if (before != (uint32_t)(r.parts - 1)) return false;
        p.arrivals[r.pair] = 0;   // for the next launch
        return true;
    };
    if (*abort_flag) {
        // nothing is written: the code says why
    } else if (warp == PRODUCER) {
        // ------------------------------------------------------------------------------------------------- producer
        const bool leader = elect_one();
        long long seq_u0 = s_start->before;
        uint32_t given = 0;        // lane w: units that warp w has been given
        uint32_t records = 0;
        int next = 0;              // the warp whose turn it is
        bool ok = true;
        // the first sequence is known; those behind it are read 32 at a time
        for (int b0 = s_start->b; b0 < p.batch && u < end && ok; b0 += 32) {
            const bool known = b0 == s_start->b;
            const int len_l = b0 + lane < p.batch ? length_of(p, b0 + lane) : 0, sh_l = b0 + lane < p.batch ? shared_of(p, b0 + lane) : 0;
            for (int i = 0; i < 32 && b0 + i < p.batch && u < end && ok; i++) {
                const int b = b0 + i;
                int len, shared;
                if (known && i == 0) {   // its units come before the others' lengths are there
                    len = s_start->len;
                    shared = s_start->shared;
                } else {
                    len = __shfl_sync(0xffffffffu, len_l, i);
                    shared = __shfl_sync(0xffffffffu, sh_l, i);
                }
                const Span x(p, len, shared);
                if (x.n == 0) continue;
                for (int kvh = u > seq_u0 ? (int)min(quotient(u - seq_u0, x.n), (long long)p.hkv) : 0; kvh < p.hkv && u < end && ok; kvh++) {
                    const long long pair_u0 = seq_u0 + (long long)kvh * x.n;
                    // (lengths that change meanwhile, which the header forbids, may leave u and pair_u0 anywhere: what is addressed by them is the pair's, or a place of a CTA of this launch in the
                    // workspace; results are wrong, and arrivals that fit no number of pieces are not zero for the stream's next call)
                    const int c_begin = (int)min(max(u - pair_u0, 0LL), (long long)x.n), c_end = (int)min((long long)x.n, c_begin + (end - u)), units = c_end - c_begin;
                    if (units == 0) continue;
                    const bool whole = units == x.n, alone = units <= ALONE, direct = whole && alone;
                    const int pair = b * p.hkv + kvh, first_warp = next, warps = alone ? 1 : min(units, CONSUMERS), record = records % RECORDS;
                    int entry = 0, entries_from = c_begin;   // lane i: the table's entry for unit entries_from + i
                    auto entries = [&](int from) {
                        const int ci = from + lane, key = (ci < x.head_units ? ci : ci + x.skip) * C::UNIT;
                        entry = -1;
                        if (ci < c_end && key < x.len) entry = __ldcg(p.block_table + (size_t)b * p.max_pages + p.page.div((uint32_t)key));
                    };
                    if (p.block_table) entries(c_begin);   // on its way beside what follows
                    if (!direct) {
                        ok = mbar_wait_warp(taken + 8 * record, (records / RECORDS & 1) ^ 1, abort_flag, ST_STREAM_LOAD);
                        if (!ok) break;
                        Pieces::Span in = {0, 1};
                        if (!whole) in = cut.pieces_of(pair_u0, x.n, gridDim.x);
                        if (leader) {
                            const uint32_t at = base + C::OFF_RECORD + 32 * record;
                            sts128(at, pair, first_warp, warps, whole ? WHOLE : u + units < end ? PIECE : TAIL);
                            sts128(at + 16, 2 * blockIdx.x + (c_begin == 0 ? 1 : 0), in.count, 2 * in.first + 1, 0);
                            mbar_arrive_count(handed + 8 * record, CONSUMERS + 1 - warps);
                        }
                        records++;
                    }
                    for (int c = c_begin; c < c_end; c++) {
                        if (p.block_table && c - entries_from >= 32) {
                            entries_from = c;
                            entries(c);
                        }
                        const int key0 = (c < x.head_units ? c : c + x.skip) * C::UNIT;
                        int row = key0, z = pair;
                        if (p.block_table) {
                            const int page = __shfl_sync(0xffffffffu, entry, c - entries_from);
                            row = key0 - (int)p.page.div((uint32_t)key0) * p.page_size;
                            z = (uint32_t)page < (uint32_t)p.num_pages ? page * p.hkv + kvh : -1;   // -1: outside the map, which arrives as zeros
                        }
                        const uint32_t nth = __shfl_sync(0xffffffffu, given, next), stage = next * DEPTH + nth % DEPTH;
                        ok = mbar_wait_warp(empty + 8 * stage, (nth / DEPTH & 1) ^ 1, abort_flag, ST_STREAM_LOAD);
                        if (!ok) break;
                        if (leader) {
                            const bool starts = alone ? c == c_begin : c - c_begin < CONSUMERS, ends = alone ? c == c_end - 1 : c + CONSUMERS >= c_end;
                            const uint32_t at = base + C::OFF_INFO + 32 * stage, bar = full + 8 * stage, q_bytes = starts ? (uint32_t)p.group * D : 0u;
                            sts128(at, key0, x.len, x.lo, x.head);
                            sts128(at + 16, (starts ? FIRST : 0) | (ends ? LAST : 0) | (direct ? DIRECT : 0), pair, record, 0);
                            mbar_arrive_expect_tx(bar, 2 * C::BYTES + q_bytes);
                            tma_load_3d(base + stage * C::BYTES, &tmap_k, bar, 0, row, z);
                            tma_load_3d(base + C::OFF_V + stage * C::BYTES, &tmap_v, bar, 0, row, z);
                            if (q_bytes) bulk_load(base + C::OFF_Q + stage * C::ROWS * D, p.q + (size_t)pair * q_bytes, q_bytes, bar);
                        }
                        given += lane == next;
                        if (!alone || c == c_end - 1) next = next + 1 < CONSUMERS ? next + 1 : 0;
                        __syncwarp();
                    }
                    u += units;
                }
                seq_u0 += (long long)x.n * p.hkv;
            }
        }
        // to everyone, that there is no more
        for (int w = 0; w < CONSUMERS && ok; w++) {
            const uint32_t nth = __shfl_sync(0xffffffffu, given, w), stage = w * DEPTH + nth % DEPTH;
            ok = mbar_wait_warp(empty + 8 * stage, (nth / DEPTH & 1) ^ 1, abort_flag, ST_STREAM_LOAD);
            if (ok && leader) {
                sts128(base + C::OFF_INFO + 32 * stage + 16, 0, NO_MORE, 0, 0);
                mbar_arrive(full + 8 * stage);
            }
        }
        if (ok && mbar_wait_warp(taken + 8 * (records % RECORDS), (records / RECORDS & 1) ^ 1, abort_flag, ST_STREAM_LOAD) && leader) {
            sts128(base + C::OFF_RECORD + 32 * (records % RECORDS), NO_MORE, 0, 0, 0);
            mbar_arrive_count(handed + 8 * (records % RECORDS), CONSUMERS + 1);
        }
    } else if (warp < CONSUMERS) {
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
        // this lane's bytes of a tile at the swizzle's places: rows g and g + 8 of K, rows 2t, 2t + 1, 2t + 8 and 2t + 9 of V (a tile's rows are a multiple of the pattern)
        auto k_at = [&](int h) -> uint32_t { return g * D + (D == 128 ? ((2 * t + h) ^ g) << 4 : (t ^ ((g >> 1) & 3)) << 4); };
        auto v_at = [&](int odd) -> uint32_t {
            const int row = 2 * t + odd;
            return row * D + (D == 128 ? (g ^ row) << 4 : (((g >> 1) ^ ((row >> 1) & 3)) << 4) + 8 * (g & 1));
        };
        uint32_t qf[NQ][C::KW];
        float m[NQ][2], l[NQ][2], acc[NQ][C::MT][4];
        uint32_t states = 0;   // that this warp has left in shared memory
        for (uint32_t nth = 0;; nth++) {
            const int stage = warp * DEPTH + nth % DEPTH;
            if (!mbar_wait_warp(full + 8 * stage, nth / DEPTH & 1, abort_flag, ST_STREAM_USE)) break;
            const Info& info = *reinterpret_cast<const Info*>(smem + C::OFF_INFO + 32 * stage);
            const int4 seen = *reinterpret_cast<const int4*>(&info.key0), what = *reinterpret_cast<const int4*>(&info.flags);
            const int flags = what.x, pair = what.y, record = what.z;
            if (pair < 0) break;
            if (flags & FIRST) {
                const uint32_t qb = base + C::OFF_Q + stage * C::ROWS * D + (D / 4) * t;
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
            const int key0 = seen.x;
            const bool cut = key0 + C::UNIT > seen.y || (key0 < seen.z && key0 + C::UNIT > seen.w);
            auto sees = [&](int key) { return key < seen.y && (key >= seen.z || key < seen.w); };
            const uint32_t kb = base + stage * C::BYTES, vb = base + C::OFF_V + stage * C::BYTES;
            // sc[n][i][e]: key g (e < 2) or g + 8 of tile i, query 8n + 2t + (e & 1)
            float sc[NQ][C::TILES][4];
#pragma unroll
            for (int i = 0; i < C::TILES; i++) {
                uint32_t kr[2][C::KW];
#pragma unroll
                for (int r = 0; r < 2; r++)
#pragma unroll
                    for (int h = 0; h < D / 64; h++) lds128(kr[r] + 4 * h, kb + (16 * i + 8 * r) * D + k_at(h));
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
                        sc[n][i][e] = x * scale_log2;
                    }
                }
            }
            if (cut) {
#pragma unroll
                for (int i = 0; i < C::TILES; i++)
#pragma unroll
                    for (int e = 0; e < 4; e += 2)
                        if (!sees(key0 + 16 * i + g + 4 * e))
#pragma unroll
                            for (int n = 0; n < NQ; n++) sc[n][i][e] = sc[n][i][e + 1] = -INFINITY;
            }
            float mx[NQ][2];
            bool bump = false;
#pragma unroll
            for (int n = 0; n < NQ; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    mx[n][e] = fmaxf(sc[n][0][e], sc[n][0][e + 2]);
#pragma unroll
                    for (int i = 1; i < C::TILES; i++) mx[n][e] = fmaxf(mx[n][e], fmaxf(sc[n][i][e], sc[n][i][e + 2]));
                    bump = bump || mx[n][e] > m[n][e] + LAG;
                }
            if (__any_sync(0xffffffffu, bump)) {   // rare once a few units are in
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
#pragma unroll
            for (int i = 0; i < C::TILES; i++) {
                uint32_t vr[4][C::VW];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const uint32_t at = vb + (16 * i + 8 * (r >> 1)) * D + v_at(r & 1);
                    if (D == 128) lds128(vr[r], at);
                    else lds64(vr[r], at);
                }
                if (i == C::TILES - 1) {   // all that the stage holds is in registers
                    __syncwarp();
                    if (lane == 0) mbar_arrive(empty + 8 * stage);
                }
                if (cut) {   // keys that are not seen may hold anything: their values must not meet a weight of zero
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (!sees(key0 + 16 * i + 2 * t + (r & 1) + 8 * (r >> 1)))
#pragma unroll
                            for (int w = 0; w < C::VW; w++) vr[r][w] = 0u;
                }
                uint32_t pf[NQ][2];   // P^T: rows (keys) 2t, 2t + 1 and 2t + 8, 2t + 9 of column g
#pragma unroll
                for (int n = 0; n < NQ; n++) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        w[e] = sc[n][i][e] == -INFINITY ? 0.f : exp2_fast(sc[n][i][e] - m[n][e & 1]);
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

            // ---- this warp's state of the pair: its O, or one of several to be added up
            if (!(flags & DIRECT)) {
                if (!mbar_wait_warp(freed + 8 * warp, (states & 1) ^ 1, abort_flag, ST_STREAM_USE)) break;
                states++;
            }
#pragma unroll
            for (int n = 0; n < NQ; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], o);
                    const int row = 8 * n + 2 * t + e;
                    if (row >= p.group) continue;
                    if (!(flags & DIRECT)) {
                        if (g == 0) s_ml[warp * C::ROWS + row] = make_float2(m[n][e], l[n][e]);
#pragma unroll
                        for (int j = 0; j < C::MT; j++) *reinterpret_cast<float2*>(&s_o[warp * C::ROWS + row][(D / 8) * g + 2 * j]) = make_float2(acc[n][j][e], acc[n][j][e + 2]);
                    } else {   // an eighth of a row to a lane
                        const size_t at = (size_t)pair * p.group + row;
#pragma unroll
                        for (int j = 0; j < C::MT; j += 2) {
                            State x;
                            x.m = m[n][e];
                            x.l = l[n][e];
                            x.o = make_float4(acc[n][j][e], acc[n][j][e + 2], acc[n][j + 1][e], acc[n][j + 1][e + 2]);
                            store_row<D>(p, at, (D / 8) * g + 2 * j, x, vds);
                        }
                    }
                }
            if (!(flags & DIRECT)) {
                __syncwarp();
                if (lane == 0) mbar_arrive(handed + 8 * record);
            }
        }
    } else {
        // ---------------------------------------------------------------- states of pairs, while the next ones are attended to
        const float vds = p.sv ? p.v_descale * ld_f32(p.sv) : p.v_descale;
        for (uint32_t nth = 0;; nth++) {
            const int slot = nth % RECORDS;
            if (!mbar_wait_warp(handed + 8 * slot, nth / RECORDS & 1, abort_flag, ST_STREAM_FINISH)) break;
            const Record r = *reinterpret_cast<const Record*>(smem + C::OFF_RECORD + 32 * slot);
            if (r.pair < 0) break;
            if (r.kind == TAIL) {   // nothing comes behind it: all warps do it, below
                if (lane == 0) left[1] = r;
            } else {
                for (int i = lane; i < p.group * (D / 4); i += 32) add_states(r, i, vds);
                __syncwarp();
                if (lane < r.count) mbar_arrive(freed + 8 * ((r.first_warp + lane) % CONSUMERS));
                if (lane == 0 && r.kind == PIECE && last_of(r)) left[0] = r;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(taken + 8 * slot);
        }
    }
    __syncthreads();
    if (*abort_flag == 0 && (left[0].parts || left[1].parts)) {
        const float vds = p.sv ? p.v_descale * ld_f32(p.sv) : p.v_descale;
        if (left[1].parts) {
            for (int i = threadIdx.x; i < p.group * (D / 4); i += THREADS) add_states(left[1], i, vds);
            __syncthreads();
            if (threadIdx.x == 0) *s_last = last_of(left[1]);
            __syncthreads();
        }
#pragma unroll 1
        for (int k = 0; k < 2; k++) {
            const Record r = left[k];
            if (r.parts == 0 || (k == 1 && !*s_last)) continue;
            for (int i = threadIdx.x; i < p.group * (D / 4); i += THREADS) {
                const int row = i / (D / 4), col = i % (D / 4) * 4;
                State x;   // slots: first_slot, then the even ones of the CTAs behind
                x.add_all<D>(p.ws_ml, p.ws_o, r.parts, col, [&](int j) { return (size_t)(j == 0 ? r.first_slot : r.first_slot + 2 * j - 1) * C::ROWS + row; });
                store_row<D>(p, (size_t)r.pair * p.group + row, col, x, vds);
            }
        }
    }
    const uint32_t code = *abort_flag;
    if (code != 0) {
        if (threadIdx.x == 0) atomicCAS(p.status, 0u, code);
        for (int i = 0; i < 200; i++) __nanosleep(1000);   // let copies already in flight land
    }
}

int unit_of(const StreamArgs& a) { return a.hd == 128 ? Cfg<128, 1>::UNIT : Cfg<64, 1>::UNIT; }
// units that a pair can have at most
long long most_units(const StreamArgs& a) {
    const long long unit = unit_of(a), all = ((long long)(a.seq_lens ? a.s_max : a.seq_len) + unit - 1) / unit;
    if (a.shared_lens) return all > 0 ? all : 1;
    const long long seen = a.window > 0 ? ((long long)a.sinks + unit - 1) / unit + ((long long)a.window + unit - 1) / unit + 1 : all;
    return seen < all ? seen : all;
}
int rows_of(const StreamArgs& a) { return a.q_heads / a.kv_heads <= 8 ? 8 : 16; }
int grid_of(const StreamArgs& a) {
    const double units = (double)most_units(a) * a.batch * a.kv_heads;
    const double resident = sms_of_current_device() * (rows_of(a) == 8 ? Cfg<128, 1>::CTAS : Cfg<128, 2>::CTAS), parts = (double)MAX_PARTS * a.batch * a.kv_heads;
    const double most = units < resident ? units : resident;
    return most < 1 ? 1 : (int)(most < parts ? most : parts);
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
    if (!make_tmap_u8_3d(&k, a.k_cache, outer, rows, a.hd, unit_of(a), a.hd, swizzle) || !make_tmap_u8_3d(&v, a.v_cache, outer, rows, a.hd, unit_of(a), a.hd, swizzle)) return cudaErrorInvalidValue;
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
