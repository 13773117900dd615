// fa_decode_fp4_sm100.cu — attention of one new token per sequence over a KV cache held in 4 bits (fa_decode_fp4,
// include/fa_sm120.h), grouped-query heads, for NVIDIA B200 (sm_100a).
//
//   o[h] = sum_k p_k V[k] / sum_k p_k,  p_k = exp(scale q[h].K[k]),  K[k][d] = code * block scale[d / 16] * tensor scale
//
// A key costs 2 * (D/2 + D/16) bytes per kv head and 4 * D flop per query head: the step is bound by the stream of the cache, and
// what it takes to keep up is few instructions per byte, for a byte is two values here.  As in the kernel over e4m3 codes
// (fa_decode_sm100.cu) codes go from global memory straight into MMA fragments, with the contraction and row indices permuted so
// that every lane's share of a row is contiguous:
//
//  * S^T = K Q^T and O^T += V^T P^T are m16n8k16 products in fp16 (16 keys, or 16 dims, are the rows, the query heads of the kv head
//    the columns).  One instruction turns two e2m1 codes into fp16 (cvt.rn.f16x2.e2m1x2 runs at the rate of an fp16 FMA: 9.5 clocks
//    for eight codes and the four FMAs that use them, of which the FMAs and a loop's add are 8.9), one multiplies them by their block scale.  Code times block
//    scale has 6 significant bits and is exact; the tensor scales go into the softmax scale and the output.
//  * The codes of V come as dims of one key, the product wants keys of one dim: the nibbles of two keys are interleaved ahead of the
//    conversion (two shifts and two bit selections for sixteen codes), so that no transposition is left.  The scales of values lie 16 keys side by side
//    in the cache for the same reason: four keys' scales are one load, and in pairs as the conversion gives them.
//  * Row g of a tile of S^T is key 4 (g / 2) + g % 2, row g + 8 the key two further: lane t of V then has keys 4t .. 4t + 3.
//  * P is kept in fp16 at up to 2^14 (a shift of 2^SHIFT, a maximum that may lag by 2^LAG): a weight keeps its 11 bits down to 2^-22 of the largest.
//
// How the keys are divided (Plan below): a CTA takes a pair (sequence, kv head), or the chunks of all pairs form one line that is cut into equal pieces.
// Pieces of a cut pair leave their states in a workspace and the CTA that finishes last adds them up in a fixed order: results do not depend on timing.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "fa_scratch_call.h"
#include "pdl.cuh"

namespace {

using namespace sm100;

constexpr int CHUNK = 64;        // keys per unit of work (page sizes are multiples of it)
constexpr int THREADS = 128;
constexpr int WARPS = THREADS / 32;
constexpr float LAG = 6.0f, SHIFT = 8.0f;   // log2 units
constexpr int ctas_per_sm(int nq) { return nq == 2 ? 2 : 3; }

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
// read once: not kept in L1
__device__ __forceinline__ void ldg128(uint32_t* r, const uint8_t* p) {
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "l"(p));
}
__device__ __forceinline__ void ldg64(uint32_t* r, const uint8_t* p) {
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "l"(p));
}
__device__ __forceinline__ uint32_t ldg32(const uint8_t* p) {
    uint32_t r;
    asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(r) : "l"(p));
    return r;
}
__device__ __forceinline__ uint32_t ldg16(const uint8_t* p) {
    uint16_t r;
    asm volatile("ld.global.L1::no_allocate.u16 %0, [%1];" : "=h"(r) : "l"(p));
    return r;
}
__device__ __forceinline__ uint32_t ldg8(const uint8_t* p) {
    uint16_t r;
    asm volatile("ld.global.L1::no_allocate.u8 %0, [%1];" : "=h"(r) : "l"(p));
    return r;
}

// Plans.
//  PAIR:  a CTA to a pair.
//  LINE:  the chunks of all pairs form one line that is cut into equal pieces, one per resident CTA, so sequences of very different
//         lengths load all SMs alike.
enum Plan : int { PAIR, LINE };

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
    // partial states, two slots per CTA: [slot][rows][D] un-normalised outputs, then [slot][rows][2] (m in log2 units, l)
    float* ws_o;
    float* ws_ml;
    uint32_t* arrivals;   // [batch * hkv], zero before and after every launch
};

template <int D, int NQ, int T>
struct Cfg {
    static constexpr int KW = D / 32;      // 32-bit words of a lane's share of one K row (eight codes each)
    static constexpr int VW = D / 64;      // the same of one V row
    static constexpr int KSTEPS = D / 16;
    static constexpr int MT = D / 16;      // 16-row tiles of O^T
    static constexpr int ROWS = 8 * NQ;    // query columns
    static constexpr int PITCH = D + 4;    // floats per row of the merge buffer
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

struct Segment {
    int b, kvh, len;                // sequence, kv head, keys of the sequence
    int n_chunks, c_begin, c_end;   // chunks of the pair, and those of them this CTA takes
    int pair_u0;                    // unit of the line where the pair starts
};

// N consecutive dims of a query, from dim d on, in fp32
template <int N>
__device__ __forceinline__ void load_q(const Params& p, size_t at, float* x) {
    if (p.q_type == FA_Q_E4M3) {
        const uint8_t* q = static_cast<const uint8_t*>(p.q) + at;
#pragma unroll
        for (int i = 0; i < N; i += 16) {
            const uint4 v = ld128(q + i);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t h = e4m3x2_to_h2(j & 1 ? w[j / 2] >> 16 : w[j / 2]);
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
                x[i + 2 * j] = f.x;
                x[i + 2 * j + 1] = f.y;
            }
        }
    } else {
        const uint16_t* q = static_cast<const uint16_t*>(p.q) + at;
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            const uint4 v = ld128(q + i);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
                if (p.q_type == FA_Q_BF16) f = make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
                x[i + 2 * j] = f.x;
                x[i + 2 * j + 1] = f.y;
            }
        }
    }
}

// T: 16-key tiles of a warp's step, which are contiguous; a CTA's step is T chunks
template <int D, int NQ, int T, bool PAGED>
__global__ void __launch_bounds__(THREADS, ctas_per_sm(NQ)) fa_decode_fp4_kernel(const Params p) {
    using C = Cfg<D, NQ, T>;
    __shared__ __align__(16) float s_o[WARPS][C::ROWS][C::PITCH];
    __shared__ float s_m[WARPS][C::ROWS], s_l[WARPS][C::ROWS];
    __shared__ Segment s_next[WARPS];
    __shared__ uint32_t s_last;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;              // MMA fragment coordinates

    // a sequence with no visible key is on nobody's piece: O = 0, LSE = -inf
    auto empty_sequence = [&](int b) {
        for (int i = 0; i < p.hq * D; i++) p.o[(size_t)b * p.hq * D + i] = __float2half_rn(0.f);
        if (p.lse)
            for (int i = 0; i < p.hq; i++) p.lse[(size_t)b * p.hq + i] = -INFINITY;
    };

    // Every warp adds the lengths up for itself (no barrier); lane i keeps those of sequences i, i + 32, .. of the first 32 * LENS, larger
    // batches read theirs again where they need them.
    constexpr int LENS = 4;
    int lens[LENS] = {};
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
    // kernel runs gets wrong results, and an empty part where the line has become shorter than u).
    auto segment_at = [&](int u, int end) {
        Segment x;
        x.b = x.kvh = x.len = x.n_chunks = x.c_begin = x.c_end = x.pair_u0 = 0;
        for (int b0 = 0, before = 0; b0 < p.batch; b0 += 32) {
            const int len = lane_len(b0), n = chunks_of(len) * p.hkv;
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
                x.kvh = (u - seq_u0) / x.n_chunks;
                x.pair_u0 = seq_u0 + x.kvh * x.n_chunks;
                x.c_begin = u - x.pair_u0;
                x.c_end = min(x.n_chunks, x.c_begin + (end - u));
                break;
            }
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
        return x;
    };

    auto page_of = [&](int key) -> int { return (int)(__umulhi((uint32_t)key, p.page_mul) >> (p.page_shr - 1)); };
    // row of the cache at which chunk c starts (the same in all four arrays; a multiple of 16), or -1 where the table names no page of
    // the pool: nothing is read there, the keys count as zeros
    auto row_of = [&](const Segment& x, int c, int page) -> long long {
        if (!PAGED) return ((long long)x.b * p.hkv + x.kvh) * p.s_max + (long long)c * CHUNK;
        if (page < 0 || page >= p.num_pages) return -1;
        const int key = c * CHUNK;
        return ((long long)page * p.hkv + x.kvh) * p.page_size + (key - page_of(key) * p.page_size);
    };

    pdl_wait();
    pdl_trigger();
    Segment seg;
    seg.b = seg.kvh = seg.len = seg.n_chunks = seg.c_begin = seg.c_end = seg.pair_u0 = 0;
    Cut cut{0, 0};
    int mid = 0, mid_end = 0;    // units of the segments still to come
    const bool line = p.plan == LINE;
    if (!line) {
        seg.b = blockIdx.x / p.hkv;
        seg.kvh = blockIdx.x - seg.b * p.hkv;
        seg.len = seq_len_of(p, seg.b);
        seg.n_chunks = seg.c_end = chunks_of(seg.len);
        if (seg.n_chunks == 0 && seg.kvh == 0 && threadIdx.x == 0) empty_sequence(seg.b);
    } else {
#pragma unroll
        for (int i = 0; i < LENS; i++) lens[i] = 32 * i + lane < p.batch ? seq_len_of(p, 32 * i + lane) : 0;
        int total = 0;
        for (int b0 = 0; b0 < p.batch; b0 += 32) {
            const int b = b0 + lane, n = chunks_of(lane_len(b0));
            if (n == 0 && b < p.batch && warp == 0 && b % gridDim.x == blockIdx.x) empty_sequence(b);
            total += __reduce_add_sync(0xffffffffu, n);
        }
        total *= p.hkv;
        const int pieces = gridDim.x;
        cut.q = total / pieces;
        cut.r = total - cut.q * pieces;
        mid = cut.begin(blockIdx.x);
        mid_end = cut.begin(blockIdx.x + 1);
        if (mid < mid_end) seg = segment_at(mid, mid_end);
        mid += seg.c_end - seg.c_begin;
    }
    if (seg.c_begin >= seg.c_end) return;
    float scale_log2 = p.scale_log2;
    if (p.sq) scale_log2 *= ld_f32(p.sq);
    if (p.sk) scale_log2 *= ld_f32(p.sk);

    // A CTA step is T chunks; tile i of warp w: keys 16i.. of the warp's own contiguous run of 16 T keys.
    const int my_chunk = (warp * T * 16) / CHUNK, my_key = (warp * T * 16) % CHUNK;
    static_assert(T <= 4, "a warp's run lies in one chunk");
    // lane-constant places inside a tile
    const int k_row = 4 * (g >> 1) + (g & 1);           // and the row two further
    const uint32_t k_lane = k_row * (D / 2) + (D / 8) * t, v_lane = 4 * t * (D / 2) + (D / 16) * g;
    const uint32_t ks_lane = k_row * (D / 16) + (D / 64) * t, vs_lane = (D == 128 ? g : g >> 1) * 16 + 4 * t;
    uint32_t kr[T][2][C::KW], ksr[T][2];                // [tile][row k_row / k_row + 2][words], scale bytes of that row
    uint32_t vr[T][4][C::VW], vsr[T];                   // [tile][keys 4t ..][words], their scale bytes
    auto entry = [&](const Segment& x, int c) -> int {   // table entry of chunk c
        return PAGED && c < x.c_end ? ld_s32(p.block_table + (size_t)x.b * p.max_pages + page_of(c * CHUNK)) : 0;
    };
    auto load_k_row = [&](int i, int r, long long row) {
        const uint8_t* codes = p.k + row * (D / 2) + (k_lane + 2 * r * (D / 2));
        const uint8_t* scales = p.ks + row * (D / 16) + (ks_lane + 2 * r * (D / 16));
        if (D == 128) ldg128(kr[i][r], codes);
        else ldg64(kr[i][r], codes);
        ksr[i][r] = D == 128 ? ldg16(scales) : ldg8(scales);
    };
    // left: keys from the chunk's first one to the end of the sequence.  Keys past it are not read but taken as zeros: they
    // may hold anything (0 x NaN would poison O)
    auto load_k = [&](int i, int left, long long row) {
        const int key = my_key + 16 * i;
#pragma unroll
        for (int r = 0; r < 2; r++) {
            if (left < CHUNK) {
#pragma unroll
                for (int w = 0; w < C::KW; w++) kr[i][r][w] = 0u;
                ksr[i][r] = 0u;
            }
            if (left >= CHUNK || key + k_row + 2 * r < left) load_k_row(i, r, row + key);
        }
    };
    auto load_v = [&](int i, int left, long long row) {
        const int key = my_key + 16 * i;
        const uint8_t* codes = p.v + (row + key) * (D / 2) + v_lane;
        const uint8_t* scales = p.vs + (row + key) * (D / 16) + vs_lane;
        const int mine = left >= CHUNK ? 4 : min(max(left - key - 4 * t, 0), 4);   // keys of this lane
        if (left < CHUNK) {
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int w = 0; w < C::VW; w++) vr[i][r][w] = 0u;
            vsr[i] = 0u;
        }
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (left >= CHUNK || r < mine) {
                if (D == 128) ldg64(vr[i][r], codes + r * (D / 2));
                else vr[i][r][0] = ldg32(codes + r * (D / 2));
            }
        if (left >= CHUNK || mine > 0) {
            vsr[i] = ldg32(scales);
            if (left < CHUNK && mine < 4) vsr[i] &= (1u << (8 * mine)) - 1u;
        }
    };
    // keys left of chunk c of a segment for load_k / load_v: none past the segment's end or where there is no page
    auto left_of = [&](const Segment& x, int c, long long row) { return c < x.c_end && row >= 0 ? x.len - c * CHUNK : 0; };

    bool loaded = false;   // the segment's first chunks are already on their way
    for (;;) {             // one segment per trip
        int page_next;
        if (!loaded) {
            const int c = seg.c_begin + my_chunk;
            const long long row = row_of(seg, c, entry(seg, c));
            const int left = left_of(seg, c, row);
#pragma unroll
            for (int i = 0; i < T; i++) {
                load_k(i, left, row);
                load_v(i, left, row);
            }
        }
        loaded = false;
        page_next = entry(seg, seg.c_begin + T + my_chunk);

        // the segment behind this one waits in shared memory (a copy per warp: no barrier)
        bool more;
        int next_entry = 0;
        {
            Segment next;
            more = line && mid < mid_end;
            if (more) {
                next = segment_at(mid, mid_end);
                more = next.c_begin < next.c_end;
                mid += next.c_end - next.c_begin;
            }
            if (more) {
                next_entry = entry(next, next.c_begin + my_chunk);
                if (lane == 0) s_next[warp] = next;
            }
            __syncwarp();
        }

        const int b = seg.b, kvh = seg.kvh;
        // Q^T fragments: dims (D/4) t + 4 ks .. + 3 of query head g of a column tile, scaled by a power of two that brings the row's largest value to
        // 2^14 .. 2^15 (no bit of bf16 is lost, and what fp16 drops lies 2^-39 below that value)
        uint32_t qf[NQ][C::KSTEPS][2];
        float f_col[NQ][2];   // score factors of query columns 2t and 2t + 1
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            float x[D / 4];
            const int row = 8 * n + g;
            if (row < p.group) {
                load_q<D / 4>(p, ((size_t)b * p.hq + (size_t)kvh * p.group + row) * D + (D / 4) * t, x);
            } else {
#pragma unroll
                for (int i = 0; i < D / 4; i++) x[i] = 0.f;
            }
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < D / 4; i++) top = fmaxf(top, fabsf(x[i]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = min(max((int)(__float_as_uint(top) >> 23), 28), 254);   // biased; what is smaller than 2^-99 counts as that
            const float up = __uint_as_float((uint32_t)(127 + 127 + 14 - e) << 23), down = __uint_as_float((uint32_t)(e - 14) << 23);
#pragma unroll
            for (int ks = 0; ks < C::KSTEPS; ks++) {
                qf[n][ks][0] = pack_h2(x[4 * ks] * up, x[4 * ks + 1] * up);
                qf[n][ks][1] = pack_h2(x[4 * ks + 2] * up, x[4 * ks + 3] * up);
            }
#pragma unroll
            for (int j = 0; j < 2; j++) f_col[n][j] = __shfl_sync(0xffffffffu, down, 4 * (2 * t + j)) * scale_log2;
        }

        // online-softmax state for query columns 2t and 2t + 1 of every column tile: running maximum less SHIFT (the same in all lanes g) and
        // this lane's part of the sum
        float m[NQ][2], l[NQ][2];
        float acc[NQ][C::MT][4];
#pragma unroll
        for (int n = 0; n < NQ; n++) {
#pragma unroll
            for (int e = 0; e < 2; e++) { m[n][e] = -INFINITY; l[n][e] = 0.f; }
#pragma unroll
            for (int i = 0; i < C::MT; i++) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.f;
        }

        for (int c = seg.c_begin; c < seg.c_end; c += T) {
            // ---- S^T = K Q^T, two accumulators: half as long a chain
            float s[NQ][T][4];
#pragma unroll
            for (int i = 0; i < T; i++) {
                uint32_t sc[2][D / 64];   // [row][group of 16 dims], in both halves
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    if (D == 128) {
                        const uint32_t pair = e4m3x2_to_h2(ksr[i][r]);
                        sc[r][0] = __byte_perm(pair, 0, 0x1010);
                        sc[r][D / 64 - 1] = __byte_perm(pair, 0, 0x3232);
                    } else {
                        sc[r][0] = e4m3x2_to_h2(ksr[i][r] * 0x0101u);
                    }
                }
                float part[NQ][2][4] = {};
#pragma unroll
                for (int w = 0; w < C::KW; w++) {
                    uint32_t x[4], y[4];
                    e2m1x8_to_h2x4(kr[i][0][w], x);
                    e2m1x8_to_h2x4(kr[i][1][w], y);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        x[j] = mul_h2(x[j], sc[0][w / 2]);
                        y[j] = mul_h2(y[j], sc[1][w / 2]);
                    }
#pragma unroll
                    for (int n = 0; n < NQ; n++)
#pragma unroll
                        for (int h = 0; h < 2; h++)
                            mma_f16_m16n8k16(part[n][h], x[2 * h], y[2 * h], x[2 * h + 1], y[2 * h + 1], qf[n][2 * w + h][0], qf[n][2 * w + h][1]);
                }
#pragma unroll
                for (int n = 0; n < NQ; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[n][i][e] = (part[n][0][e] + part[n][1][e]) * f_col[n][e & 1];
            }
            // ---- the next chunks' keys, of this segment or, behind its last ones, of the next: the merge below then hides
            // their latency
            const bool roll = c + T >= seg.c_end;
            const bool fetch = !roll || more;
            int left_n = 0;
            long long row_n = -1;
            if (!roll) {
                const int cn = c + T + my_chunk;
                row_n = row_of(seg, cn, page_next);
                left_n = left_of(seg, cn, row_n);
                page_next = entry(seg, cn + T);
            } else if (more) {
                const Segment next = s_next[warp];
                const int cn = next.c_begin + my_chunk;
                row_n = row_of(next, cn, next_entry);
                left_n = left_of(next, cn, row_n);
                loaded = true;
            }
            if (fetch) {
#pragma unroll
                for (int i = 0; i < T; i++) load_k(i, left_n, row_n);
            }
            // ---- softmax and O^T += V^T P^T, 16 keys at a time.  s[n][i][e] = key k_row (e < 2) or k_row + 2 of tile i, query 8n + 2t + (e & 1)
            const int ci = c + my_chunk, key_end = ci < seg.c_end ? seg.len : 0;
#pragma unroll
            for (int i = 0; i < T; i++) {
                const int key0 = ci * CHUNK + my_key + 16 * i;
                if (key0 + 16 > key_end) {   // only the last chunk of a sequence has keys past its end
#pragma unroll
                    for (int n = 0; n < NQ; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (key0 + k_row + 2 * (e >> 1) >= key_end) s[n][i][e] = -INFINITY;
                }
                float mx[NQ][2];
                bool bump = false;
#pragma unroll
                for (int n = 0; n < NQ; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        mx[n][e] = fmaxf(s[n][i][e], s[n][i][e + 2]) - SHIFT;
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
                            const float f = m[n][e] == -INFINITY ? 1.f : ex2f(m[n][e] - m_new);   // nothing but NaN has been added where there is no maximum
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
                uint32_t pf[NQ][2];
#pragma unroll
                for (int n = 0; n < NQ; n++) {
                    float pv[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        pv[e] = s[n][i][e] == -INFINITY ? 0.f : ex2f(s[n][i][e] - m[n][e & 1]);
                        l[n][e & 1] += pv[e];
                    }
                    pf[n][0] = transpose_8x8_b16(pack_h2(pv[0], pv[1]));
                    pf[n][1] = transpose_8x8_b16(pack_h2(pv[2], pv[3]));
                }
                // rows g and g + 8 of tile j of O^T are d = (D/8) g + 2j and + 1
                const uint32_t s01 = e4m3x2_to_h2(vsr[i]), s23 = e4m3x2_to_h2(vsr[i] >> 16);
#pragma unroll
                for (int w = 0; w < C::VW; w++) {
                    uint32_t a[4][4];   // even and odd dims of keys 0 and 1, and of 2 and 3
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t x = vr[i][2 * h][w], y = vr[i][2 * h + 1][w];
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
                        for (int n = 0; n < NQ; n++) mma_f16_m16n8k16(acc[n][4 * w + j], a[0][j], a[1][j], a[2][j], a[3][j], pf[n][0], pf[n][1]);
                    }
                }
            }
            if (fetch) {
#pragma unroll
                for (int i = 0; i < T; i++) load_v(i, left_n, row_n);
            }
        }

        // ---- merge the four warps' states
        const bool whole = seg.c_begin == 0 && seg.c_end == seg.n_chunks;
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], o);
                const int row = 8 * n + 2 * t + e;
                if (g == 0) {
                    s_m[warp][row] = m[n][e];
                    s_l[warp][row] = l[n][e];
                }
                if (row < p.group) {
#pragma unroll
                    for (int j = 0; j < C::MT; j++)
                        *reinterpret_cast<float2*>(&s_o[warp][row][(D / 8) * g + 2 * j]) = make_float2(acc[n][j][e], acc[n][j][e + 2]);
                }
            }
        __syncthreads();
        // slots of a cut pair: the odd slot of the CTA that has its first piece and the even slots of the CTAs after that
        const int slot = 2 * blockIdx.x + (seg.c_begin == 0 ? 1 : 0);
        const float vds = p.sv ? p.v_descale * ld_f32(p.sv) : p.v_descale;
        for (int idx = threadIdx.x; idx < p.group * (D / 4); idx += THREADS) {   // four columns per thread and step
            const int row = idx / (D / 4), col = idx % (D / 4) * 4;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; w++) M = fmaxf(M, s_m[w][row]);
            float L = 0.f;
            float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                const float mw = s_m[w][row];
                fold(L, O, s_l[w][row], *reinterpret_cast<const float4*>(&s_o[w][row][col]), mw == -INFINITY ? 1.f : ex2f(mw - M));
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
            // the pair's pieces: slot0, then slot0 + 1 + 2 i
            const int first = cut.piece_of(seg.pair_u0), parts = cut.piece_of(seg.pair_u0 + seg.n_chunks - 1) - first + 1, slot0 = 2 * first + 1;
            const int bh = b * p.hkv + kvh;
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                s_last = atomicAdd(p.arrivals + bh, 1u) == (uint32_t)(parts - 1);
                if (s_last) p.arrivals[bh] = 0;   // for the next launch
            }
            __syncthreads();
            if (s_last) {
                __threadfence();
                for (int idx = threadIdx.x; idx < p.group * (D / 4); idx += THREADS) {
                    const int row = idx / (D / 4), col = idx % (D / 4) * 4;
                    float M = -INFINITY, L = 0.f;
                    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int i0 = 0; i0 < parts; i0 += 8) {   // eight pieces' loads in flight
                        float2 ml[8];
                        float4 oi[8];
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            const int i = i0 + k;
                            ml[k] = make_float2(-INFINITY, 0.f);
                            oi[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (i >= parts) continue;
                            const size_t at = (size_t)(i == 0 ? slot0 : slot0 + 1 + (i - 1) * 2) * C::ROWS + row;
                            ml[k] = __ldcg(reinterpret_cast<const float2*>(p.ws_ml + at * 2));
                            oi[k] = __ldcg(reinterpret_cast<const float4*>(p.ws_o + at * D + col));
                        }
                        float M2 = M;
#pragma unroll
                        for (int k = 0; k < 8; k++) M2 = fmaxf(M2, ml[k].x);
                        const float f = M == -INFINITY ? 1.f : ex2f(M - M2);
                        L *= f;
                        O.x *= f; O.y *= f; O.z *= f; O.w *= f;
#pragma unroll
                        for (int k = 0; k < 8; k++) fold(L, O, ml[k].y, oi[k], ml[k].x == -INFINITY ? 1.f : ex2f(ml[k].x - M2));
                        M = M2;
                    }
                    store_out<D>(p, ((size_t)b * p.hq + (size_t)kvh * p.group + row), col, M, L, O, vds);
                }
            }
        } else {
            __syncthreads();   // the merge buffer is free again
        }
        if (!more) break;
        seg = s_next[warp];
        __syncwarp();
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

struct Layout {
    int plan, grid, rows;
};
// A CTA to a pair once the pairs nearly fill the SMs and sequences are short, or there are several pairs to a resident CTA: a piece of a cut
// pair costs some microseconds of latency that nothing hides.  And where a line had more chunks than an int counts (a paged cache whose
// capacity is far above what it holds).
Layout layout_of(int batch, int q_heads, int kv_heads, int span) {
    Layout x;
    x.rows = q_heads / kv_heads <= 8 ? 8 : 16;
    const long long pairs = (long long)batch * kv_heads, chunks = ((long long)span + CHUNK - 1) / CHUNK;
    const long long resident = (long long)ctas_per_sm(x.rows / 8) * num_sms_of_current_device();
    if (2 * pairs >= (x.rows == 8 ? 6 : 3) * resident || (chunks <= 32 && 5 * pairs >= 4 * resident) || pairs * chunks > 0x7fffffffLL) {
        x.plan = PAIR;
        x.grid = (int)pairs;
    } else {
        x.plan = LINE;
        const long long units = pairs * chunks;
        x.grid = (int)(units < resident ? (units > 0 ? units : 1) : resident);
    }
    return x;
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
    p.ws_ml = p.ws_o + (size_t)c.x.grid * 2 * c.x.rows * c.hd;
    p.arrivals = scratch.zeros;
    auto run = [&](auto contiguous, auto paged) { return launch_pdl(p.block_table ? paged : contiguous, dim3((unsigned)c.x.grid), dim3(THREADS), 0, c.stream, p); };
#define KERNEL(D, NQ, T) run(fa_decode_fp4_kernel<D, NQ, T, false>, fa_decode_fp4_kernel<D, NQ, T, true>)
    if (c.x.rows == 8) return c.hd == 64 ? KERNEL(64, 1, 4) : KERNEL(128, 1, 2);
    return c.hd == 64 ? KERNEL(64, 2, 4) : KERNEL(128, 2, 2);
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
    if (s_max % 16 != 0) return refuse(ctx, who, FA_ERR_INVALID_ARG, "s_max must be a multiple of 16");
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
    c.x = layout_of(g->batch, g->q_heads, g->kv_heads, span);
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
    return fa_sm100::call_with_scratch(ctx, who, c.stream, cuts ? (size_t)c.x.grid * c.x.rows * 2 * (c.hd + 2) * sizeof(float) : 0,
                                       cuts ? (size_t)g->batch * g->kv_heads : 0, launch, &c);
}
