// fa_decode_fp4_sm100.cu — attention of one new token per sequence over a KV cache held in 4 bits (fa_decode_fp4,
// include/fa_sm120.h), grouped-query heads, for NVIDIA B200 (sm_100a).
//
//   o[h] = sum_k p_k V[k] / sum_k p_k,  p_k = exp(scale q[h].K[k]),  K[k][d] = code * block scale[d / 16] * tensor scale
//
// A key costs 2 * (D/2 + D/16) bytes per kv head and 4 * D flop per query head: the step is bound by the stream of the cache, and what it takes to keep up is few
// instructions per byte, for a byte is two values here.  16 keys of 128 dims, 2304 bytes, are 262 instructions of a warp; the memory's rate leaves time for about 390.  116 of them
// are for the pipe of conversions and logic (64 conversions of code pairs, 16 that sort V's codes), which takes one in two clocks: 232 clocks of a quadrant.
//
//  * S^T = K Q^T and O^T += V^T P^T are m16n8k16 products in fp16 (16 keys, or 16 dims, are the rows, the query heads of the kv head the columns; two column tiles for
//    groups of 9 to 16), with contraction and row indices permuted so that every lane's share of a row is contiguous.  One instruction turns two e2m1 codes into fp16
//    (2.2 clocks of a quadrant, as much as one fp16x2 multiplication), one multiplies them by their block scale.  Code times block scale has 6 significant bits and is
//    exact; the tensor scales go into the softmax scale and the output.
//  * The codes of V come as dims of one key, the product wants keys of one dim: the nibbles of two keys are interleaved ahead of the conversion (two shifts and two
//    bit selections for sixteen codes), so that no transposition is left.  The scales of values lie 16 keys side by side in the cache for the same reason: four
//    keys' scales are one load, and in pairs as the conversion gives them.
//  * Row g of a tile of S^T is key 4 (g / 2) + g % 2, row g + 8 the key two further: lane t of V then has keys 4t .. 4t + 3.
//  * A warp has a ring of stages of 64 keys in shared memory that it fills for itself by asynchronous copies, across the ends of pairs.  (Codes from global memory straight
//    into registers, as the kernel over e4m3 codes has them, left no registers for enough bytes in flight: 64 sequences of 2048 to 4096 keys, 32 heads, 304 us, with the
//    ring 186.)  Three CTAs to an SM, whose warps add their states up in the stage that the
//    last step has read and take the products of two tiles side by side, are ahead of two with four (64 sequences of 1024 to 4096 keys, 32 heads, 150 / 157 us; of two column tiles
//    three spill), and steps of 64 keys of 32 (155 / 161).
//  * P is kept in fp16 at up to 2^14: a weight keeps its 11 bits down to 2^-28 of the largest, and the largest is 2^14 itself, so that a key that outweighs the others loses nothing.  (A
//    maximum that lags spares steps and is 1 % faster, but O of rows that one key dominates is then off by that key's rounding: 1.6 times as far as its own rounding to fp16 puts it, for 1.2.)
//
// How the keys are divided (fa_decode_fp4_layout.h, and Teams below): pieces of a cut pair leave their states in a workspace and the team that hands in the last one adds them up in a
// fixed order: results do not depend on timing.
//
// Measured: 64 sequences of 3000 keys, 32 heads of 128, 150 us = 5.9 TB/s of cache (0.90 of the rate of a copy; 175 at 1.72 GHz after a second of it, under the power cap); 8 kv heads of
// 4 query heads 4.4 TB/s (256 sequences of 1000 keys) and 5.2 (of 2000), 4 of 16 2.5 (100 of 1500); 4 kv heads of 64, 4 query heads each, 4.1 (400 of 1200; a key's softmax is the same for half
// the bytes), 16 each 1.8 (48 of 2250).
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "fa_decode_fp4_layout.h"
#include "fa_scratch_call.h"
#include "pdl.cuh"

namespace {

using namespace fa_fp4;
using namespace sm100;

constexpr int PIECES = 8;        // pieces of a pair whose loads are in flight at once
constexpr int MANY = 16;         // pieces of a pair from which on sums of eight are formed first
constexpr float SHIFT = 14.0f;   // log2 units

__device__ __forceinline__ void mma_f16_m16n8k16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8_b16(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// two at a time: a = a * f + c, and a += b
__device__ __forceinline__ void fma_x2(float& a0, float& a1, float f0, float f1, float c0, float c1) {
    asm("{\n\t.reg .b64 a, f, c;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 f, {%2, %3};\n\tmov.b64 c, {%4, %5};\n\tfma.rn.f32x2 a, a, f, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "+f"(a0), "+f"(a1)
        : "f"(f0), "f"(f1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void add_x2(float& a0, float& a1, float b0, float b1) {
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}" : "+f"(a0), "+f"(a1) : "f"(b0), "f"(b1));
}
// the bytes of w, two e2m1 codes each -> four fp16 pairs (low code in the low half)
__device__ __forceinline__ void e2m1x8_to_h2x4(uint32_t w, uint32_t* h) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}
// the low two bytes of w, e4m3 -> an fp16 pair
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t w) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(w));
    return r;
}
// 16 bytes from global to shared memory past L1
__device__ __forceinline__ void copy16(uint32_t to, const uint8_t* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// the first `bytes` of them, and zeros for the others
__device__ __forceinline__ void copy16(uint32_t to, const uint8_t* from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {   // all but the last N groups are there
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

struct Params {
    const void* q;
    const uint8_t *k, *ks, *v, *vs;
    __half* o;
    float* lse;
    const int* seq_lens;
    int q_type, batch, hq, hkv, group, s_max, seq_len;
    float scale_log2, v_descale;
    const float *sq, *sk, *sv;
    int plan;
    // paged cache: the chunk at key k0 of sequence b lies in page block_table[b * max_pages + k0 / page_size]
    const int* block_table;
    int page_size, max_pages, num_pages;
    uint32_t page_mul, page_shr;   // key / page_size as multiply-high and shift
    // partial states, two slots per team and behind those two per eight teams: [slot][rows][D] un-normalised outputs, then [slot][rows][2] (m in log2 units, l)
    float* ws_o;
    float* ws_ml;
    uint32_t* arrivals;   // [batch * hkv] and two for every eight teams, zero before and after every launch
};

constexpr int T = 4;   // 16-key tiles of a warp's step: a chunk
template <int D, int NQ>
struct Cfg {
    static constexpr int KW = D / 32;      // 32-bit words of a lane's share of one K row (eight codes each)
    static constexpr int VW = D / 64;      // the same of one V row
    static constexpr int KSTEPS = D / 16;
    static constexpr int MT = D / 16;      // 16-row tiles of O^T
    static constexpr int ROWS = 8 * NQ;    // query columns
    static constexpr int PITCH = D + 4;    // floats per row of the merge buffer
    // a stage of a warp's ring: codes of K and of V, block scales of K and of V, of 16 T keys
    static constexpr int CODES = 16 * T * D / 2, SCALES = 16 * T * D / 16, STAGE = 2 * (CODES + SCALES);
    static constexpr int STAGES = D == 128 ? 2 : 3;
    static constexpr int RING_BYTES = WARPS * STAGES * STAGE;
};

__device__ __forceinline__ int seq_len_of(const Params& p, int b) { return p.seq_lens ? min(max(__ldcg(p.seq_lens + b), 0), p.s_max) : p.seq_len; }
__device__ __forceinline__ int chunks_of(int len) { return (len + CHUNK - 1) / CHUNK; }

// [begin, end) of piece i of equal pieces of a line (the first `remainder` pieces are one unit longer), and back
struct Cut {
    int q, r;
    __device__ __forceinline__ int begin(int i) const { return i * q + min(i, r); }
    __device__ __forceinline__ int piece_of(int u) const { return u < r * (q + 1) ? u / (q + 1) : r + (u - r * (q + 1)) / q; }
};

__device__ __forceinline__ void fold(float& L, float4& O, float l, const float4& o, float f) {
    L += l * f;
    O.x += o.x * f; O.y += o.y * f; O.z += o.z * f; O.w += o.w * f;
}
template <int D>
__device__ __forceinline__ void store_out(const Params& p, size_t row, int col, float M, float L, const float4& O, float vds) {
    const float inv = L == 0.f ? 0.f : vds / L;   // a NaN stays one
    if ((reinterpret_cast<uintptr_t>(p.o) & 7) == 0) {   // o need only be 2-byte aligned
        *reinterpret_cast<uint2*>(p.o + row * D + col) = make_uint2(pack_h2(O.x * inv, O.y * inv), pack_h2(O.z * inv, O.w * inv));
    } else {
        __half* h = p.o + row * D + col;
        h[0] = __float2half_rn(O.x * inv); h[1] = __float2half_rn(O.y * inv);
        h[2] = __float2half_rn(O.z * inv); h[3] = __float2half_rn(O.w * inv);
    }
    if (col == 0 && p.lse) p.lse[row] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}

// one more at a counter, behind what the team has written and ahead of what it reads; how many there were
__device__ __forceinline__ uint32_t arrive(uint32_t* counter) {
    uint32_t n;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(n) : "l"(counter) : "memory");
    return n;
}

struct Segment {
    int b, kvh, len;                // sequence, kv head, keys of the sequence
    int n_chunks, c_begin, c_end;   // chunks of the pair, and those of them this team takes
    int pair_u0, u_end;             // units of the line where the pair's chunks start and where this part ends
};

// A lane's share of a query, D / 4 dims from (D / 4) t on: as it lies in memory, and as numbers
template <int D>
struct RawQ {
    uint4 w[D / 32];   // 8 values of 16 bits each; of e4m3 the first half
};
template <int D>
__device__ __forceinline__ void load_q(const Params& p, int b, int head, int t, RawQ<D>& r) {
    const size_t at = ((size_t)b * p.hq + head) * D + (D / 4) * t;
    const uint8_t* q = static_cast<const uint8_t*>(p.q) + (p.q_type == FA_Q_E4M3 ? at : 2 * at);
#pragma unroll
    for (int i = 0; i < D / 32; i++)
        if (i < D / 64 || p.q_type != FA_Q_E4M3) r.w[i] = ld128(q + 16 * i);
}
template <int D>
__device__ __forceinline__ void values_of(int q_type, const RawQ<D>& r, float* x) {
    uint32_t w[D / 8];
#pragma unroll
    for (int i = 0; i < D / 32; i++) { w[4 * i] = r.w[i].x; w[4 * i + 1] = r.w[i].y; w[4 * i + 2] = r.w[i].z; w[4 * i + 3] = r.w[i].w; }
#pragma unroll
    for (int j = 0; j < D / 8; j++) {
        const uint32_t h = q_type == FA_Q_E4M3 ? e4m3x2_to_h2(j & 1 ? w[j / 2] >> 16 : w[j / 2]) : w[j];
        float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        if (q_type == FA_Q_BF16) f = make_float2(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u));
        x[2 * j] = f.x;
        x[2 * j + 1] = f.y;
    }
}

// Teams.  A team is what a piece of the line, or a pair, is given to: the CTA, whose warps take runs of 16 T keys of a step in turn and add their states up in the end, or
// (ALONE) each of its warps.
template <int D, int NQ, bool ALONE, bool PAGED>
__global__ void __launch_bounds__(THREADS, ctas_per_sm(NQ)) fa_decode_fp4_kernel(const Params p) {
    using C = Cfg<D, NQ>;
    __shared__ float s_m[WARPS][C::ROWS], s_l[WARPS][C::ROWS];
    __shared__ uint32_t s_last[WARPS];
    extern __shared__ __align__(128) uint8_t s_ring[];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;              // MMA fragment coordinates
    constexpr int TEAM = ALONE ? 1 : WARPS, TEAMS = WARPS / TEAM, TEAM_THREADS = 32 * TEAM;
    constexpr int STEP = 16 * T * TEAM, STEP_CHUNKS = TEAM;   // keys of a team's step
    static_assert(16 * T == CHUNK, "a warp's run of a step is a chunk");
    const int team = ALONE ? warp : 0, rank = ALONE ? 0 : warp, thread = ALONE ? lane : threadIdx.x;   // the latter two in the team
    const int me = blockIdx.x * TEAMS + team, pieces = gridDim.x * TEAMS;
    auto team_sync = [&] {
        if (ALONE) __syncwarp();
        else __syncthreads();
    };

    // O = 0 and LSE = -inf for query heads of a sequence with no visible key
    auto no_keys = [&](int b, int head, int heads) {
        const size_t row = (size_t)b * p.hq + head;
        for (int i = thread; i < heads * (D / 4); i += TEAM_THREADS) store_out<D>(p, row + i / (D / 4), i % (D / 4) * 4, -INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f), 0.f);
    };

    // Every warp adds the lengths up for itself (no barrier); lane i keeps those of sequences i, i + 32, .. of the first 32 * LENS, larger
    // batches read theirs again where they need them.
    constexpr int LENS = 4;
    int lens[LENS] = {};
    int per_lane = 1, units_to = 0;   // groups of 32 sequences of a lane, and units of all sequences' first kv heads up to the end of its own
    auto lane_len = [&](int b0) -> int {   // length of sequence b0 + lane, b0 a multiple of 32
        if (b0 < 32 * LENS) {
            int x = lens[0];
#pragma unroll
            for (int i = 1; i < LENS; i++)
                if (b0 == 32 * i) x = lens[i];
            return x;
        }
        return b0 + lane < p.batch ? seq_len_of(p, b0 + lane) : 0;
    };
    // the part of one pair that starts at unit u and ends at unit end or with the pair.  The sequence, its length and what lies before it
    // come from one reading of the lengths: nothing is addressed from two that disagree (a caller that rewrites them while the
    // kernel runs, which the header forbids, gets wrong results, an empty part where the line has become shorter than u, and arrivals that fit no team's count: counters that
    // are not zero for the stream's next call).
    auto units_of = [&](int len) -> int { return len > 0 ? chunks_of(len) + pair_cost<ALONE>(chunks_of(len)) : 0; };
    auto segment_at = [&](int u, int end) {
        Segment x;
        x.b = x.kvh = x.len = x.n_chunks = x.c_begin = x.c_end = x.pair_u0 = 0;
        x.u_end = end;
        const uint32_t lanes = __ballot_sync(0xffffffffu, units_to * p.hkv > u);   // the first of these has the groups where it lies
        if (lanes == 0) return x;
        const int of = __ffs(lanes) - 1, units_before = __shfl_sync(0xffffffffu, units_to, max(of - 1, 0));
        for (int b0 = 32 * per_lane * of, before = of ? units_before * p.hkv : 0; b0 < min(p.batch, 32 * per_lane * (of + 1)); b0 += 32) {
            const int len = lane_len(b0), n = units_of(len) * p.hkv;
            int incl = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, before + incl > u);   // first lane whose sequence ends past u
            if (past) {
                const int at = __ffs(past) - 1, seq_u0 = before + __shfl_sync(0xffffffffu, incl - n, at);
                x.b = b0 + at;
                x.len = __shfl_sync(0xffffffffu, len, at);
                x.n_chunks = chunks_of(x.len);
                const int units = units_of(x.len);
                x.kvh = (u - seq_u0) / units;
                x.pair_u0 = seq_u0 + x.kvh * units + (units - x.n_chunks);
                x.u_end = min(end, x.pair_u0 + x.n_chunks);
                x.c_begin = max(u - x.pair_u0, 0);
                x.c_end = x.u_end - x.pair_u0;   // nothing where the piece ends ahead of the first chunk
                break;
            }
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
        return x;
    };

    auto page_of = [&](int key) -> int { return (int)(__umulhi((uint32_t)key, p.page_mul) >> (p.page_shr - 1)); };
    pdl_wait();
    pdl_trigger();
    const float f_q = p.sq ? ld_f32(p.sq) : 1.f, f_k = p.sk ? ld_f32(p.sk) : 1.f, f_v = p.sv ? ld_f32(p.sv) : 1.f;   // on their way while the piece is found
    Segment seg;
    seg.b = seg.kvh = seg.len = seg.n_chunks = seg.c_begin = seg.c_end = seg.pair_u0 = seg.u_end = 0;
    Cut cut{0, 0};
    int mid_end = 0;    // unit of the line where this team's piece ends
    const bool line = p.plan == LINE;
    if (!line) {
        seg.b = me / p.hkv;
        seg.kvh = me - seg.b * p.hkv;
        if (seg.b >= p.batch) return;
        seg.len = seq_len_of(p, seg.b);
        seg.n_chunks = seg.c_end = chunks_of(seg.len);
        if (seg.n_chunks == 0) no_keys(seg.b, seg.kvh * p.group, p.group);
    } else {
#pragma unroll
        for (int i = 0; i < LENS; i++) lens[i] = 32 * i + lane < p.batch ? seq_len_of(p, 32 * i + lane) : 0;
        const int groups = (p.batch + 31) / 32;
        per_lane = (groups + 31) / 32;
#pragma unroll 4
        for (int i = 0; i < groups; i++) {
            const int n = units_of(lane_len(32 * i));
            const uint32_t empty = __ballot_sync(0xffffffffu, n == 0 && 32 * i + lane < p.batch && (32 * i + lane) % pieces == me);
            const int sum = __reduce_add_sync(0xffffffffu, n);
            if (lane == i / per_lane) units_to += sum;
            // a sequence that is empty is on nobody's piece
            for (uint32_t x = empty; x; x &= x - 1) no_keys(32 * i + __ffs(x) - 1, 0, p.hq);
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, units_to, o);
            if (lane >= o) units_to += y;
        }
        const int total = __shfl_sync(0xffffffffu, units_to, 31) * p.hkv;
        cut.q = total / pieces;
        cut.r = total - cut.q * pieces;
        const int begin = cut.begin(me);
        mid_end = cut.begin(me + 1);
        if (begin < mid_end) seg = segment_at(begin, mid_end);
    }
    if (seg.c_begin >= seg.c_end) return;
    // the part behind one, empty where there is none
    auto next_of = [&](const Segment& x) {
        if (line && x.u_end < mid_end) {
            if (x.kvh + 1 == p.hkv) return segment_at(x.u_end, mid_end);
            Segment y = x;   // the same sequence's next kv head
            y.kvh++;
            y.pair_u0 += units_of(x.len);
            y.u_end = min(mid_end, y.pair_u0 + y.n_chunks);
            y.c_begin = 0;
            y.c_end = y.u_end - y.pair_u0;
            return y;
        }
        Segment none = x;
        none.c_begin = none.c_end = 0;
        return none;
    };
    // queries of a part
    RawQ<D> raw_q[NQ];
    auto ask_q = [&](const Segment& x) {
#pragma unroll
        for (int n = 0; n < NQ; n++)
            if (8 * n + g < p.group) load_q<D>(p, x.b, x.kvh * p.group + 8 * n + g, t, raw_q[n]);
    };
    ask_q(seg);   // ahead of the stream of keys, behind which they would wait

    // A warp takes a contiguous run of 16 T keys of a step, and has a ring of stages of its own for them, filled by copies of its own: no barrier but the warp's.
    // Rows are stored 16 bytes by 16, at places of a 128-byte line that are exchanged by a pattern of the line's number such that the
    // reads of K (rows k_row of eight lanes g) and of V (rows 4t + r of four lanes t) meet no bank twice.
    const int my_chunk = rank;
    uint8_t* const ring = s_ring + warp * C::STAGES * C::STAGE;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    const int k_row = 4 * (g >> 1) + (g & 1);           // and the row two further
    // places inside a tile
    const uint32_t k_at = D == 128 ? (g >> 1) * 256 + ((((g & 1) * 4 + t) ^ ((g >> 1) << 1)) * 16)
                                   : (g >> 1) * 128 + ((((g & 1) * 2 + (t >> 1)) ^ (((g >> 1) & 1) << 2 | ((g >> 1) & 2))) * 16) + (t & 1) * 8;
    const uint32_t v_at = D == 128 ? 2 * t * 128 + (((g >> 1) ^ (t << 1)) * 16) + (g & 1) * 8 : t * 128 + (((g >> 2) ^ ((t & 1) << 2 | (t & 2))) * 16) + (g & 3) * 4;
    const uint32_t ks_at = k_row * (D / 16) + (D / 64) * t, vs_at = (D == 128 ? g : g >> 1) * 16 + 4 * t;
    const uint32_t put_at = (lane >> 3) * 128 + (D == 128 ? ((lane & 7) ^ ((lane >> 4) << 1)) * 16 : ((lane & 7) ^ (((lane >> 3) & 1) << 2 | ((lane >> 3) & 2))) * 16);

    // What is to be fetched next: a part, steps of it that are left, keys from the run's first one to the end of what the part's sequence has.  Places in the cache
    // are counted in blocks of 16 rows (of which there are fewer than 2^32 in any memory); of a paged one every lane has that of one of 32 steps, made from table
    // entries asked for 32 steps before.
    constexpr uint32_t NO_PAGE = 0xffffffffu;
    Segment f_seg;
    int f_steps, f_left, f_step = 0;
    uint32_t f_block = 0, f_blocks = 0, f_to = ring_at;
    int f_entry = 0;
    auto left_of = [&](const Segment& x) { return min(x.len, x.c_end * CHUNK) - (x.c_begin + my_chunk) * CHUNK; };
    auto steps_of = [&](const Segment& x) { return (x.c_end - x.c_begin + STEP_CHUNKS - 1) / STEP_CHUNKS; };
    auto entry = [&](int c) -> int {   // table entry of the lane's step of the 32 from chunk c on
        c += my_chunk + STEP_CHUNKS * lane;
        return c < f_seg.c_end ? ld_s32(p.block_table + (size_t)f_seg.b * p.max_pages + page_of(c * CHUNK)) : -1;
    };
    auto begin_fetch = [&](const Segment& x) {
        f_seg = x;
        f_steps = steps_of(x);
        f_left = left_of(x);
        f_step = 0;
        if (PAGED) f_entry = f_steps > 0 ? entry(x.c_begin) : -1;
        else f_block = ((uint32_t)x.b * p.hkv + x.kvh) * (uint32_t)(p.s_max / 16) + (x.c_begin + my_chunk) * (CHUNK / 16);
    };
    constexpr int CODE_COPIES = C::CODES / 512, SCALE_PIECES = C::SCALES / 16, SCALE_COPIES = (2 * SCALE_PIECES + 31) / 32;
    static_assert(SCALE_COPIES <= 2 && (SCALE_COPIES == 1 || SCALE_PIECES == 32), "a lane's scale copies are of keys or of values");
    auto of_values = [&](int j) { return 32 * j + lane >= SCALE_PIECES; };
    const uint8_t* const from_k = p.k + lane * 16;
    const uint8_t* const from_v = p.v + lane * 16;
    const uint8_t* from_scales[SCALE_COPIES];
#pragma unroll
    for (int j = 0; j < SCALE_COPIES; j++) from_scales[j] = of_values(j) ? p.vs + (32 * j + lane - SCALE_PIECES) * 16 : p.ks + (32 * j + lane) * 16;
    const bool has_scales = 2 * SCALE_PIECES >= 32 || lane < 2 * SCALE_PIECES;
    auto fetch = [&] {
        if (f_steps > 0) {
            if (PAGED) {
                if (f_step == 0) {
                    const int c = (min(f_seg.len, f_seg.c_end * CHUNK) - f_left) / CHUNK;   // the warp's chunk
                    const int key = (c + STEP_CHUNKS * lane) * CHUNK;
                    f_blocks = f_entry >= 0 && f_entry < p.num_pages
                                   ? ((uint32_t)f_entry * p.hkv + f_seg.kvh) * (uint32_t)(p.page_size / 16) + (uint32_t)(key - page_of(key) * p.page_size) / 16
                                   : NO_PAGE;
                    f_entry = entry(c - my_chunk + 32 * STEP_CHUNKS);
                }
                f_block = __shfl_sync(0xffffffffu, f_blocks, f_step);
                f_step = (f_step + 1) & 31;
            }
            // Keys past the sequence's end are not read but taken as zeros: they may hold anything (0 x NaN would poison O).  So are all where there is no page.
            if (f_left > 0) {
                const int left = PAGED && f_block == NO_PAGE ? 0 : f_left;
                const uint32_t to = f_to + put_at, to_odd = D == 128 ? to ^ 64 : to, to_scales = f_to + 2 * C::CODES + lane * 16;
                const uint8_t *k = from_k + (size_t)f_block * (8 * D), *v = from_v + (size_t)f_block * (8 * D);
                if (left >= 16 * T) {
#pragma unroll
                    for (int j = 0; j < CODE_COPIES; j++) copy16((j & 1 ? to_odd : to) + j * 512, k + j * 512);
#pragma unroll
                    for (int j = 0; j < CODE_COPIES; j++) copy16((j & 1 ? to_odd : to) + C::CODES + j * 512, v + j * 512);
#pragma unroll
                    for (int j = 0; j < SCALE_COPIES; j++)
                        if (has_scales) copy16(to_scales + j * 512, from_scales[j] + (size_t)f_block * D);
                } else {
                    constexpr int ROWS_OF_COPY = 1024 / D, LANES_OF_ROW = D / 32;
#pragma unroll
                    for (int j = 0; j < CODE_COPIES; j++) {
                        const bool there = ROWS_OF_COPY * j + lane / LANES_OF_ROW < left;
                        copy16((j & 1 ? to_odd : to) + j * 512, there ? k + j * 512 : p.k, there ? 16 : 0);
                        copy16((j & 1 ? to_odd : to) + C::CODES + j * 512, there ? v + j * 512 : p.v, there ? 16 : 0);
                    }
#pragma unroll
                    for (int j = 0; j < SCALE_COPIES; j++) {
                        const int i = 32 * j + lane;
                        // of keys 256 / D rows to 16 bytes, of values 16 keys
                        const int bytes = min(max(of_values(j) ? left - (i - SCALE_PIECES) / (D / 16) * 16 : (left - i * (256 / D)) * (D / 16), 0), 16);
                        if (has_scales) copy16(to_scales + j * 512, bytes ? from_scales[j] + (size_t)f_block * D : p.ks, bytes);
                    }
                }
            }
            f_to = f_to + C::STAGE == ring_at + C::STAGES * C::STAGE ? ring_at : f_to + C::STAGE;
            if (!PAGED) f_block += STEP / 16;
            f_left -= STEP;
            if (--f_steps == 0) begin_fetch(next_of(f_seg));
        }
        copies_commit();
    };
    begin_fetch(seg);
#pragma unroll
    for (int i = 0; i < C::STAGES - 1; i++) fetch();

    int stage = 0;
    for (;;) {             // one segment per trip
        const int b = seg.b, kvh = seg.kvh;
        // Q^T fragments: dims (D/4) t + 4 ks .. + 3 of query head g of a column tile, scaled by a power of two that brings the row's largest value to
        // 2^14 .. 2^15 (no bit of bf16 is lost, and what fp16 drops lies 2^-39 below that value), and by the sign of the scale: the factor of a score is positive
        uint32_t qf[NQ][C::KSTEPS][2];
        float f_col[NQ][2];   // factors of the scores of query columns 2t and 2t + 1
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            float x[D / 4];
            values_of<D>(p.q_type, raw_q[n], x);
            if (8 * n + g >= p.group) {
#pragma unroll
                for (int i = 0; i < D / 4; i++) x[i] = 0.f;
            }
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < D / 4; i++) top = fmaxf(top, fabsf(x[i]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = min(max((int)(__float_as_uint(top) >> 23), 28), 254);   // biased; what is smaller than 2^-99 counts as that
            const float scale = p.scale_log2 * f_q * f_k;
            const float up = copysignf(__uint_as_float((uint32_t)(127 + 127 + 14 - e) << 23), scale), down = __uint_as_float((uint32_t)(e - 14) << 23);
#pragma unroll
            for (int ks = 0; ks < C::KSTEPS; ks++) {
                qf[n][ks][0] = pack_h2(x[4 * ks] * up, x[4 * ks + 1] * up);
                qf[n][ks][1] = pack_h2(x[4 * ks + 2] * up, x[4 * ks + 3] * up);
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float f = __shfl_sync(0xffffffffu, down, 4 * (2 * t + j)) * fabsf(scale);
                f_col[n][j] = f == 0.f ? 1e-38f : f;   // a hidden key's -inf stays one
            }
        }

        // online-softmax state for query columns 2t and 2t + 1 of every column tile: running maximum ahead of f_col (the same in all lanes g) and
        // this lane's part of the sum.  A weight is 2^((s - m) f_col + SHIFT): the difference first, so that none passes 2^SHIFT however large the scores are (a difference of products that
        // is rounded at once with them passes it by the product's last bits: infinite in fp16 from 2^25 on)
        float m[NQ][2], l[NQ][2];
        float acc[NQ][C::MT][4];
#pragma unroll
        for (int n = 0; n < NQ; n++) {
#pragma unroll
            for (int e = 0; e < 2; e++) { m[n][e] = -INFINITY; l[n][e] = 0.f; }
#pragma unroll
            for (int i = 0; i < C::MT; i++) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.f;
        }

        int left = left_of(seg);   // keys from the run's first to the end
        for (int step = steps_of(seg); step > 0; step--, left -= STEP) {
            copies_wait<C::STAGES - 2>();
            __syncwarp();   // all lanes' copies are there, and all lanes have read the stage before this one
            fetch();
            const uint8_t* const st = ring + stage;
            stage = stage + C::STAGE == C::STAGES * C::STAGE ? 0 : stage + C::STAGE;
            if (left <= 0) continue;
            // ---- S^T = K Q^T, several tiles side by side: a product waits for the one before it
            float s[NQ][T][4] = {};
            constexpr int SIDE = NQ == 1 && D == 64 ? T : 2;   // as many as the registers hold
#pragma unroll
            for (int i0 = 0; i0 < T; i0 += SIDE) {
                uint32_t sc[SIDE][2][D / 64];   // [row][group of 16 dims], in both halves
                uint32_t kr[SIDE][2][C::KW];
#pragma unroll
                for (int i = 0; i < SIDE; i++)
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const uint8_t* const at = st + (i0 + i) * 8 * D + (D == 128 ? k_at + r * 128 : k_at ^ (r * 64));
                        const uint8_t* const sc_at = st + 2 * C::CODES + (16 * (i0 + i) + 2 * r) * (D / 16) + ks_at;
                        if (D == 128) {
                            const uint4 x = *reinterpret_cast<const uint4*>(at);
                            kr[i][r][0] = x.x; kr[i][r][1] = x.y; kr[i][r][C::KW - 2] = x.z; kr[i][r][C::KW - 1] = x.w;
                            const uint32_t pair = e4m3x2_to_h2(*reinterpret_cast<const uint16_t*>(sc_at));
                            sc[i][r][0] = __byte_perm(pair, 0, 0x1010);
                            sc[i][r][D / 64 - 1] = __byte_perm(pair, 0, 0x3232);
                        } else {
                            const uint2 x = *reinterpret_cast<const uint2*>(at);
                            kr[i][r][0] = x.x; kr[i][r][1] = x.y;
                            sc[i][r][0] = e4m3x2_to_h2(*sc_at * 0x0101u);
                        }
                    }
#pragma unroll
                for (int w = 0; w < C::KW; w++) {
                    uint32_t x[SIDE][4], y[SIDE][4];
#pragma unroll
                    for (int i = 0; i < SIDE; i++) {
                        e2m1x8_to_h2x4(kr[i][0][w], x[i]);
                        e2m1x8_to_h2x4(kr[i][1][w], y[i]);
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            x[i][j] = mul_h2(x[i][j], sc[i][0][w / 2]);
                            y[i][j] = mul_h2(y[i][j], sc[i][1][w / 2]);
                        }
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int i = 0; i < SIDE; i++)
#pragma unroll
                            for (int n = 0; n < NQ; n++)
                                mma_f16_m16n8k16(s[n][i0 + i], x[i][2 * h], y[i][2 * h], x[i][2 * h + 1], y[i][2 * h + 1], qf[n][2 * w + h][0], qf[n][2 * w + h][1]);
                }
            }
            // ---- softmax over the step's keys.  s[n][i][e], yet to be multiplied by f_col, = key k_row (e < 2) or k_row + 2 of tile i, query 8n + 2t + (e & 1)
            if (left < 16 * T) {   // only the last chunk of a sequence has keys past its end
#pragma unroll
                for (int n = 0; n < NQ; n++)
#pragma unroll
                    for (int i = 0; i < T; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (16 * i + k_row + 2 * (e >> 1) >= left) s[n][i][e] = -INFINITY;
            }
            float mx[NQ][2];
            bool bump = false;
#pragma unroll
            for (int n = 0; n < NQ; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float x = fmaxf(s[n][0][e], s[n][0][e + 2]);
#pragma unroll
                    for (int i = 1; i < T; i++) x = fmaxf(x, fmaxf(s[n][i][e], s[n][i][e + 2]));
                    mx[n][e] = x;
                    bump = bump || x > m[n][e];
                }
            if (__any_sync(0xffffffffu, bump)) {   // rare once a few chunks are in
#pragma unroll
                for (int n = 0; n < NQ; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) mx[n][e] = fmaxf(mx[n][e], __shfl_xor_sync(0xffffffffu, mx[n][e], o));
                        const float m_new = fmaxf(m[n][e], mx[n][e]);
                        const float f = m[n][e] == -INFINITY ? 1.f : ex2f((m[n][e] - m_new) * f_col[n][e]);   // nothing but NaN has been added where there is no maximum
                        m[n][e] = m_new;
                        l[n][e] *= f;
#pragma unroll
                        for (int j = 0; j < C::MT; j++) {
                            acc[n][j][e] *= f;
                            acc[n][j][e + 2] *= f;
                        }
                    }
            }
            // P^T as B fragments: rows 2t, 2t + 1 and 2t + 8, 2t + 9, which are keys 4t .. 4t + 3, of column g
            uint32_t pf[NQ][T][2];
#pragma unroll
            for (int n = 0; n < NQ; n++) {
                // where there is no maximum yet every score is -inf (or NaN, which stays): any finite number will do for it
                const float m0 = m[n][0] == -INFINITY ? 0.f : -m[n][0], m1 = m[n][1] == -INFINITY ? 0.f : -m[n][1];
#pragma unroll
                for (int i = 0; i < T; i++) {
                    float pv[4];
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        pv[e] = s[n][i][e];
                        pv[e + 1] = s[n][i][e + 1];
                        add_x2(pv[e], pv[e + 1], m0, m1);
                        fma_x2(pv[e], pv[e + 1], f_col[n][0], f_col[n][1], SHIFT, SHIFT);
                        pv[e] = ex2f(pv[e]);
                        pv[e + 1] = ex2f(pv[e + 1]);
                        add_x2(l[n][0], l[n][1], pv[e], pv[e + 1]);
                    }
                    pf[n][i][0] = transpose_8x8_b16(pack_h2(pv[0], pv[1]));
                    pf[n][i][1] = transpose_8x8_b16(pack_h2(pv[2], pv[3]));
                }
            }
            // ---- O^T += V^T P^T: rows g and g + 8 of tile j of O^T are d = (D/8) g + 2j and + 1
#pragma unroll
            for (int i = 0; i < T; i++) {
                const uint32_t scales = *reinterpret_cast<const uint32_t*>(st + 2 * C::CODES + C::SCALES + i * D + vs_at);
                const uint32_t s01 = e4m3x2_to_h2(scales), s23 = e4m3x2_to_h2(scales >> 16);
                uint32_t vr[4][C::VW];   // keys 4t ..
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const uint8_t* const at = st + C::CODES + i * 8 * D + (D == 128 ? (v_at ^ ((r & 1) * 64)) + (r >> 1) * 128 : v_at ^ (r * 32));
                    if (D == 128) {
                        const uint2 x = *reinterpret_cast<const uint2*>(at);
                        vr[r][0] = x.x; vr[r][C::VW - 1] = x.y;
                    } else {
                        vr[r][0] = *reinterpret_cast<const uint32_t*>(at);
                    }
                }
#pragma unroll
                for (int w = 0; w < C::VW; w++) {
                    uint32_t a[4][4];   // even and odd dims of keys 0 and 1, and of 2 and 3
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t x = vr[2 * h][w], y = vr[2 * h + 1][w];
                        e2m1x8_to_h2x4((x & 0x0f0f0f0fu) | ((y << 4) & 0xf0f0f0f0u), a[2 * h]);
                        e2m1x8_to_h2x4(((x >> 4) & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u), a[2 * h + 1]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        a[0][j] = mul_h2(a[0][j], s01);
                        a[1][j] = mul_h2(a[1][j], s01);
                        a[2][j] = mul_h2(a[2][j], s23);
                        a[3][j] = mul_h2(a[3][j], s23);
#pragma unroll
                        for (int n = 0; n < NQ; n++) mma_f16_m16n8k16(acc[n][4 * w + j], a[0][j], a[1][j], a[2][j], a[3][j], pf[n][i][0], pf[n][i][1]);
                    }
                }
            }
        }

        // ---- the next part's queries; add the team's states up
        const Segment next = next_of(seg);
        const bool more = next.c_begin < next.c_end;
        if (more) ask_q(next);
        const bool whole = seg.c_begin == 0 && seg.c_end == seg.n_chunks;
        // the stage of the last step is free until the next part's first step asks for more
        static_assert(C::ROWS * C::PITCH * 4 <= C::STAGE, "a state fits a stage");
        const int free_stage = stage ? stage - C::STAGE : (C::STAGES - 1) * C::STAGE;
        auto o_at = [&](int w, int row, int col) { return reinterpret_cast<float*>(s_ring + w * C::STAGES * C::STAGE + free_stage) + row * C::PITCH + col; };
        __syncwarp();
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], o);
                const int row = 8 * n + 2 * t + e;
                if (g == 0) {
                    s_m[warp][row] = fmaf(m[n][e], f_col[n][e], -SHIFT);
                    s_l[warp][row] = l[n][e];
                }
                if (row < p.group) {
#pragma unroll
                    for (int j = 0; j < C::MT; j++)
                        *reinterpret_cast<float2*>(o_at(warp, row, (D / 8) * g + 2 * j)) = make_float2(acc[n][j][e], acc[n][j][e + 2]);
                }
            }
        team_sync();
        // slots of a cut pair: the odd slot of the team that has its first piece and the even slots of those after that
        const int slot = 2 * me + (seg.c_begin == 0 ? 1 : 0);
        const float vds = p.v_descale * f_v;
        for (int idx = thread; idx < p.group * (D / 4); idx += TEAM_THREADS) {   // four columns per thread and step
            const int row = idx / (D / 4), col = idx % (D / 4) * 4;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < TEAM; w++) M = fmaxf(M, s_m[team * TEAM + w][row]);
            float L = 0.f;
            float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = team * TEAM; w < team * TEAM + TEAM; w++) {
                const float mw = s_m[w][row];
                fold(L, O, s_l[w][row], *reinterpret_cast<const float4*>(o_at(w, row, col)), mw == -INFINITY ? 1.f : ex2f(mw - M));
            }
            if (whole) {
                store_out<D>(p, ((size_t)b * p.hq + (size_t)kvh * p.group + row), col, M, L, O, vds);
            } else {
                const size_t at = (size_t)slot * C::ROWS + row;
                __stcg(reinterpret_cast<float4*>(p.ws_o + at * D + col), O);
                if (col == 0) __stcg(reinterpret_cast<float2*>(p.ws_ml + at * 2), make_float2(M, L));
            }
        }
        if (!whole) {
            // The pair's pieces are those of teams first .. last.  The team that hands in the last one adds them up; of many, those of eight teams side by side are added
            // up by the last of these, and the sums by the last of those: a round of loads each, the first by many teams at a time.
            const int first = cut.piece_of(seg.pair_u0), last = cut.piece_of(seg.pair_u0 + seg.n_chunks - 1), pair = b * p.hkv + kvh;
            auto handed_in_last = [&](int counter, int of) {
                team_sync();   // what this team has written is written, and the merge buffer free again
                if (thread == 0) {
                    const bool is_last = arrive(p.arrivals + counter) == (uint32_t)(of - 1);
                    if (is_last) p.arrivals[counter] = 0;   // for the next launch
                    s_last[team] = is_last;
                }
                team_sync();
                return s_last[team] != 0;
            };
            // the states in `parts` slots added up
            auto add_up = [&](int parts, auto&& slot_of, auto&& put) {
                for (int idx = thread; idx < p.group * (D / 4); idx += TEAM_THREADS) {
                    const int row = idx / (D / 4), col = idx % (D / 4) * 4;
                    float M = -INFINITY, L = 0.f;
                    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int i0 = 0; i0 < parts; i0 += PIECES) {   // so many pieces' loads in flight
                        float2 ml[PIECES];
                        float4 oi[PIECES];
                        float M2 = M;
#pragma unroll
                        for (int k = 0; k < PIECES; k++) {
                            const int i = i0 + k;
                            ml[k] = make_float2(-INFINITY, 0.f);
                            oi[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (i >= parts) continue;
                            const size_t at = (size_t)slot_of(i) * C::ROWS + row;
                            ml[k] = __ldcg(reinterpret_cast<const float2*>(p.ws_ml + at * 2));
                            oi[k] = __ldcg(reinterpret_cast<const float4*>(p.ws_o + at * D + col));
                        }
#pragma unroll
                        for (int k = 0; k < PIECES; k++) M2 = fmaxf(M2, ml[k].x);
                        const float f = M == -INFINITY ? 1.f : ex2f(M - M2);
                        L *= f;
                        O.x *= f; O.y *= f; O.z *= f; O.w *= f;
#pragma unroll
                        for (int k = 0; k < PIECES; k++) fold(L, O, ml[k].y, oi[k], ml[k].x == -INFINITY ? 1.f : ex2f(ml[k].x - M2));
                        M = M2;
                    }
                    put(row, col, M, L, O);
                }
            };
            auto put_out = [&](int row, int col, float M, float L, const float4& O) { store_out<D>(p, ((size_t)b * p.hq + (size_t)kvh * p.group + row), col, M, L, O, vds); };
            auto piece = [&](int from, int i) { return 2 * (from + i) + (from + i == first ? 1 : 0); };
            // counter, and slot behind those of the pieces, of the sum of eight teams' pieces of a pair that starts before them or among them
            auto sum = [&](int eight) { return 2 * eight + (first >= 8 * eight ? 1 : 0); };
            if (last - first < MANY) {
                if (handed_in_last(pair, last - first + 1)) add_up(last - first + 1, [&](int i) { return piece(first, i); }, put_out);
            } else {
                const int eight = me / 8, from = max(first, 8 * eight), n = min(last, 8 * eight + 7) - from + 1;
                if (handed_in_last(p.batch * p.hkv + sum(eight), n)) {
                    add_up(n, [&](int i) { return piece(from, i); }, [&](int row, int col, float M, float L, const float4& O) {
                        const size_t at = (size_t)(2 * pieces + sum(eight)) * C::ROWS + row;
                        __stcg(reinterpret_cast<float4*>(p.ws_o + at * D + col), O);
                        if (col == 0) __stcg(reinterpret_cast<float2*>(p.ws_ml + at * 2), make_float2(M, L));
                    });
                    if (handed_in_last(pair, last / 8 - first / 8 + 1)) add_up(last / 8 - first / 8 + 1, [&](int i) { return 2 * pieces + sum(first / 8 + i); }, put_out);
                }
            }
        } else {
            team_sync();   // the merge buffer is free again
        }
        if (!more) break;
        seg = next;
    }
}

int num_sms_of_current_device() {
    static int cached[64];   // 0 = not asked yet; every thread would store the same value
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) != cudaSuccess) return sms;
    if (dev >= 0 && dev < 64 && cached[dev]) return cached[dev];
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (dev >= 0 && dev < 64) cached[dev] = sms;
    return sms;
}

struct Call {
    Params p;
    Layout x;
    int hd;
    cudaStream_t stream;
};

cudaError_t launch(const void* args, const fa_sm100::CallScratch& scratch) {
    const Call& c = *static_cast<const Call*>(args);
    Params p = c.p;
    p.ws_o = static_cast<float*>(scratch.workspace);
    p.ws_ml = p.ws_o + (size_t)c.x.slots() * c.x.rows * c.hd;
    p.arrivals = scratch.zeros;
    static std::atomic<bool> known[16][64];   // kernels whose shared memory has been asked for, by device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    // What fits the SMs with fewer CTAs to each asks for so much shared memory that no more share one: they would be placed three to an SM while others have one
    // (288 pairs of 4096 keys 46 us for 34).
    const int sms = num_sms_of_current_device(), spread = c.x.grid <= sms ? 116 << 10 : c.x.grid <= 2 * sms ? 80 << 10 : 0;
    auto run = [&](auto contiguous, auto paged, int ring) {
        const int smem = std::max(ring, spread), most = std::max(ring, 116 << 10);
        auto kernel = p.block_table ? paged : contiguous;
        const int which = (c.x.alone ? 8 : 0) + (c.x.rows == 16 ? 4 : 0) + (c.hd == 128 ? 2 : 0) + (p.block_table ? 1 : 0);
        if (dev >= 64 || !known[which][dev].load(std::memory_order_relaxed)) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
            if (e != cudaSuccess) return e;
            if (dev < 64) known[which][dev].store(true, std::memory_order_relaxed);
        }
        return launch_pdl(kernel, dim3((unsigned)c.x.grid), dim3(THREADS), smem, c.stream, p);
    };
#define KERNEL(D, NQ, ALONE) run(fa_decode_fp4_kernel<D, NQ, ALONE, false>, fa_decode_fp4_kernel<D, NQ, ALONE, true>, Cfg<D, NQ>::RING_BYTES)
    if (c.x.alone) {
        if (c.x.rows == 8) return c.hd == 64 ? KERNEL(64, 1, true) : KERNEL(128, 1, true);
        return c.hd == 64 ? KERNEL(64, 2, true) : KERNEL(128, 2, true);
    }
    if (c.x.rows == 8) return c.hd == 64 ? KERNEL(64, 1, false) : KERNEL(128, 1, false);
    return c.hd == 64 ? KERNEL(64, 2, false) : KERNEL(128, 2, false);
#undef KERNEL
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

}  // namespace

extern "C" fa_status_t fa_decode_fp4(fa_ctx_t* ctx, const fa_decode_fp4_args_t* g) {
    using fa_sm100::refuse;
    const char* who = "fa_decode_fp4";
    if (!ctx) return FA_ERR_INVALID_ARG;
    if (!g) return refuse(ctx, who, FA_ERR_INVALID_ARG, "null argument block");
    if (!g->q || !g->k_codes || !g->k_scales || !g->v_codes || !g->v_scales || !g->o)
        return refuse(ctx, who, FA_ERR_INVALID_ARG, "null pointer in q/k_codes/k_scales/v_codes/v_scales/o");
    if (g->q_type != FA_Q_BF16 && g->q_type != FA_Q_FP16 && g->q_type != FA_Q_E4M3) return refuse(ctx, who, FA_ERR_INVALID_ARG, "q_type must be FA_Q_BF16, FA_Q_FP16 or FA_Q_E4M3");
    const bool paged = g->block_table != nullptr;
    if (paged && (g->page_size <= 0 || g->page_size % CHUNK != 0 || g->max_pages_per_seq <= 0 || g->num_pages <= 0 ||
                  (long long)g->page_size * g->max_pages_per_seq > 0x7fffffffLL))
        return refuse(ctx, who, FA_ERR_INVALID_ARG, "paged cache needs page_size a positive multiple of 64, max_pages_per_seq > 0 and num_pages > 0");
    const int s_max = paged ? g->page_size * g->max_pages_per_seq : g->s_max;
    if (g->batch <= 0 || g->q_heads <= 0 || g->kv_heads <= 0 || s_max <= 0) return refuse(ctx, who, FA_ERR_INVALID_ARG, "batch/heads/s_max must be > 0");
    if (s_max % 16 != 0 || s_max > 0x7fffffff - (CHUNK - 1)) return refuse(ctx, who, FA_ERR_INVALID_ARG, "s_max must be a multiple of 16 and at most 2^31 - 64");
    if (g->head_dim != 64 && g->head_dim != 128) return refuse(ctx, who, FA_ERR_UNSUPPORTED_HD, "head_dim must be 64 or 128");
    if (g->q_heads % g->kv_heads != 0 || g->q_heads / g->kv_heads > 16)
        return refuse(ctx, who, FA_ERR_UNSUPPORTED_SHAPE, "q_heads must be a multiple of kv_heads with at most 16 query heads per kv head");
    if ((long long)g->batch * g->kv_heads > 0x7fffffffLL) return refuse(ctx, who, FA_ERR_UNSUPPORTED_SHAPE, "batch * kv_heads must be below 2^31");
    if (!g->seq_lens && (g->seq_len < 0 || g->seq_len > s_max)) return refuse(ctx, who, FA_ERR_INVALID_ARG, "seq_len must be in [0, s_max]");
    if (!aligned(g->q, 16) || !aligned(g->k_codes, 16) || !aligned(g->k_scales, 16) || !aligned(g->v_codes, 16) || !aligned(g->v_scales, 16) || !aligned(g->o, 2) ||
        !aligned(g->l_out, 4) || !aligned(g->seq_lens, 4) || !aligned(g->block_table, 4))
        return refuse(ctx, who, FA_ERR_INVALID_ARG, "q, codes and scales must be 16-byte aligned, lengths, table and l_out 4-byte aligned");
    const fa_status_t ok = fa_sm100::usable(ctx, who);
    if (ok != FA_OK) return ok;
    const int span = g->seq_lens ? s_max : g->seq_len;
    Call c;
    c.x = layout_of(g->batch, g->q_heads, g->kv_heads, span, paged ? (long long)g->page_size * g->num_pages : (long long)span * g->batch,
                     num_sms_of_current_device());
    c.hd = g->head_dim;
    c.stream = reinterpret_cast<cudaStream_t>(g->stream);
    Params& p = c.p;
    p = Params{};
    p.q = g->q;
    p.k = static_cast<const uint8_t*>(g->k_codes); p.ks = static_cast<const uint8_t*>(g->k_scales);
    p.v = static_cast<const uint8_t*>(g->v_codes); p.vs = static_cast<const uint8_t*>(g->v_scales);
    p.o = static_cast<__half*>(g->o);
    p.lse = static_cast<float*>(g->l_out);
    p.seq_lens = g->seq_lens;
    p.q_type = g->q_type;
    p.batch = g->batch; p.hq = g->q_heads; p.hkv = g->kv_heads; p.group = g->q_heads / g->kv_heads;
    p.s_max = s_max; p.seq_len = g->seq_len;
    p.scale_log2 = g->scale * 1.4426950408889634f;
    p.v_descale = g->v_descale == 0.0f ? 1.0f : g->v_descale;
    p.sq = g->scale_q_dev; p.sk = g->scale_k_dev; p.sv = g->scale_v_dev;
    p.plan = c.x.plan;
    p.block_table = g->block_table;
    p.page_size = g->page_size; p.max_pages = g->max_pages_per_seq; p.num_pages = g->num_pages;
    if (paged) {   // page_size >= 64; exact for numerators below 2^31, and the multiplier fits 32 bits
        uint32_t lg = 0;
        while ((1ull << lg) < (unsigned)g->page_size) lg++;
        p.page_mul = (uint32_t)(((1ull << (31 + lg)) + g->page_size - 1) / g->page_size);
        p.page_shr = lg;   // umulhi is >> 32: >> (31 + lg) is >> (lg - 1) more
    }
    const bool cuts = c.x.plan == LINE;
    return fa_sm100::call_with_scratch(ctx, who, c.stream, cuts ? (size_t)c.x.slots() * c.x.rows * (c.hd + 2) * sizeof(float) : 0,
                                       cuts ? (size_t)g->batch * g->kv_heads + c.x.sums() : 0, launch, &c);
}
