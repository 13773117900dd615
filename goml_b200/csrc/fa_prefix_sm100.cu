// fa_prefix_sm100.cu — FP8 decode attention for sequences that begin alike (fa_decode_shared; sm_100a): what they have in common is read once for all of them.
//
// The new tokens of a group's n sequences, with the g query heads that share a kv head, are n g rows that see the same keys: a product like a prompt's, and no longer one that
// reads 2 hd bytes for 4 hd g flops.  Four kernels:
//  1. fa_decode_stream_kernel (fa_decode_stream_sm100.cu): the keys that every sequence has to itself; bound by memory.
//  2. prefix_plan_kernel: beside it, one CTA finds how many pieces the groups' prefixes are cut into (128 rows of one kv head against one run of blocks of 64 keys each), so that
//     they fill the CTAs that are resident, and writes a record for each.
//  3. fa_prefix_kernel: what the sequences have in common, a piece at a time: S = Q K^T (tcgen05, e4m3) and O += P V (tcgen05, fp16: P from tensor memory, V converted in shared
//     memory) with the running maximum and sum of a softmax, a row to a thread.  A row that has less in common than others of its group sees that much of the piece.
//  4. prefix_sum_kernel: the states of every row added up.
// The roles of a CTA of the third kernel are those of the prompt's attention: four softmax warps, one that issues the products, one that loads, two that convert V; two CTAs to an SM,
// so that one's products run under the other's exponentials.  Bound by what the schedulers issue and the exponentials (16 a clock and SM), which take about as long, where rows are many.
// Measured in a CUDA graph of ten, 32 query and 8 kv heads of 128: 64 sequences behind 30000 keys 56.3 us (559 TFLOP/s of all four kernels), behind 110000 131.6 us (876): 1090 clocks of an SM for 128 rows
// against 64 keys, and some 25 us for the launches' chain, the pieces' ends and their states.  Against the kernel as it was when each was tried: eight softmax warps, half a row to a thread, took 20 % longer;
// scores of which a few left the registers 7 %; votes on every block 3 %.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/fa_sm120.h"
#include "fa_convert_v.cuh"
#include "fa_decode_mma.cuh"
#include "fa_decode_stream.h"
#include "fa_scratch_call.h"
#include "fa_softmax.cuh"
#include "pdl.cuh"
#include "row_items.cuh"
#include "sm100_ptx.cuh"
#include "tmap.cuh"

namespace fa_sm100 {

namespace {

using namespace sm100;

constexpr int BM = 128, BN = V_KEYS;      // rows of a piece, keys of a block
// Rings: memory answers after a microsecond, in which a CTA may be through with a block and a half, so codes of K and V are asked for four blocks ahead; of V in fp16 two
// tiles do.
constexpr int K_STAGES = 4, RAW_STAGES = 4, V_STAGES = 2;
constexpr int SOFTMAX_WARPS = 4, MMA_WARP = 4, LOAD_WARP = 5, CONVERT_WARP = 6, CONVERTERS = 2, THREADS = 8 * 32;
constexpr int NAN_SLOTS = 8;
constexpr int CTAS = 2;                   // of an SM
// Bytes of keys and values that sharing can save at most (all that the sequences have room for, but for a share of one sequence to each group), up to which each reads its own: what
// the three further kernels take.  The host knows the room, not the lengths, so a table that is wider than its sequences takes the kernels sooner than it should (8 behind 2000: 16.7 us, or 20.9 where there
// is room for more).  Own / shared, us, in CUDA graphs of ten on one cache, rooms as wide as the sequences (MB that sharing can save): 32 query heads, 8 kv heads of 128, behind 2000, 8 sequences 16.7 / 20.9 (30),
// 16 17.9 / 21.5 (65), 32 25.2 / 27.5 (133), 64 38.9 / 30.5 (271); 16 behind 5000 27.8 / 25.5 (157); 16 behind 2000, 32 kv heads, 37.4 / 24.8 (258); in five groups, 16 behind 8000 38.5 / 37.9 (182), 32 behind 5000 45.5
// / 35.0 (282).  The two are within 10 % from 130 to 185 MB.  Of head dim 64: 8 kv heads, behind 2000, 16 sequences 14.6 / 20.0 (32), 32 19.1 / 21.6 (67), 64 26.9 / 23.2 (135); 32 kv heads, 8 18.7 / 20.6 (60), 16 26.1 /
// 22.1 (129); one kv head, 16 query heads, behind 3000, 100 23.1 / 25.0 (39), 200 31.9 / 30.6 (79); five groups, 32 behind 5000, 29.4 / 27.5 (141).
constexpr double own_bytes(int hd) { return hd == 128 ? 1.9e8 : 1e8; }
constexpr int MAX_SPLITS = 64;            // pieces of a prefix
constexpr int MAX_GROUPS = 2048;          // whose starts, keys and first pieces the planner has in shared memory
constexpr float TAU = 6.0f, POFF = 2.0f;  // the running maximum may lag by 2^TAU; P is carried as P 2^POFF, at most 2^8
constexpr uint32_t IDESC_NEGATE_A = 1u << 13;
enum : uint32_t { ST_PREFIX_LOAD = 0x251, ST_PREFIX_MMA = 0x252, ST_PREFIX_SOFTMAX = 0x253, ST_PREFIX_CONVERT = 0x254, ST_PREFIX_SMEM = 0x255 };

struct Piece {
    int seq0, row0, rows, kvh;     // first sequence of the group; rows [row0, row0 + rows) of its (sequences x query heads of the kv head)
    int blk0, nblk, split, keys;   // blocks; which piece of the prefix; keys that the group has in common
};
// ------------------------------------------------------------------------------------------------------------------- plan
struct PlanParams {
    const int *seq_lens, *shared_lens, *starts;
    int batch, groups, group, hkv, s_max, max_splits, max_pieces, resident;
    int* pieces;      // their number
    Piece* piece;
    int* splits;      // [batch]: pieces that hold keys of a sequence
};
__device__ __forceinline__ int in_common(const PlanParams& p, int b) { return min(min(max(__ldcg(p.seq_lens + b), 0), p.s_max), max(__ldcg(p.shared_lens + b), 0)); }
__device__ __forceinline__ int blocks_of(int keys) { return keys > 0 ? (keys - 1) / BN + 1 : 0; }
__device__ __forceinline__ int at_most(long long x) { return (int)min(x, 0x3fffffffLL); }

constexpr int PLAN_THREADS = 256;
__global__ void __launch_bounds__(PLAN_THREADS) prefix_plan_kernel(const PlanParams p) {
    extern __shared__ int scratch[];   // 3 groups + 1
    __shared__ unsigned long long s_best;
    __shared__ int s_keys, sums[PLAN_THREADS / 32];
    // Nothing here comes from the kernel ahead, which has waited for all that is ahead of the two.
    pdl_trigger();
    int *const starts = scratch, *const keys = starts + p.groups + 1, *const base = keys + p.groups;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = PLAN_THREADS / 32;
    for (int i = threadIdx.x; i <= p.groups; i += PLAN_THREADS) starts[i] = min(max(__ldcg(p.starts + i), 0), p.batch);
    for (int i = threadIdx.x; i < p.groups; i += PLAN_THREADS) keys[i] = 0;
    if (threadIdx.x == 0) {
        s_best = ~0ull;
        s_keys = 0;
    }
    __syncthreads();
    // ---- keys of every group: the most that one of its sequences has in common
    int most = 0;
    for (int b = threadIdx.x; b < p.batch; b += PLAN_THREADS) {
        const int n = in_common(p, b);
        int i = 0;   // the last group that starts at or before b
        for (int step = 1 << (31 - __clz(p.groups)); step; step >>= 1)
            if (i + step <= p.groups && starts[i + step] <= b) i += step;
        if (i < p.groups && n) {
            atomicMax(keys + i, n);
            most = max(most, n);
        }
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0 && most) atomicMax(&s_keys, most);
    __syncthreads();
    const int blocks = blocks_of(s_keys);   // of the longest
    auto row_tiles = [&](int i) { return max((int)(((long long)(starts[i + 1] - starts[i]) * p.group + BM - 1) / BM), 0); };
    auto splits = [&](int i, int per) { return (blocks_of(keys[i]) + per - 1) / per; };
    auto count = [&](int i, int per) { return at_most((long long)row_tiles(i) * p.hkv * splits(i, per)); };
    // ---- blocks of a piece: rounds of the resident CTAs times what a piece takes (its start and end take as long as some eight blocks), and the states that are
    // to be added up
    for (int n = 1 + warp; n <= p.max_splits && n <= blocks; n += warps) {
        const int per = (blocks + n - 1) / n;
        long long pieces = 0;
        for (int i = lane; i < p.groups; i += 32) pieces += count(i, per);
        pieces = __reduce_add_sync(0xffffffffu, (uint32_t)min(pieces, 0x3ffffffLL));
        const unsigned long long rounds = (pieces + p.resident - 1) / p.resident, cost = rounds * (per + 8) * 2 + (blocks + per - 1) / per;
        if (lane == 0) atomicMin(&s_best, min(cost, 1ull << 37) << 26 | (unsigned)per);   // ties: the fewer blocks
    }
    __syncthreads();
    const int per = blocks ? (int)(s_best & 0x3ffffffu) : 1;
    // ---- where the pieces of a group start
    int before = 0;
    for (int i0 = 0; i0 < p.groups; i0 += PLAN_THREADS) {
        const int i = i0 + threadIdx.x, n = i < p.groups ? count(i, per) : 0;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl = at_most((long long)incl + y);
        }
        if (lane == 31) sums[warp] = incl;
        __syncthreads();
        int here = 0, all = 0;
        for (int w = 0; w < warps; w++) {
            if (w < warp) here = at_most((long long)here + sums[w]);
            all = at_most((long long)all + sums[w]);
        }
        if (i < p.groups) base[i] = at_most((long long)before + here + incl - n);
        before = at_most((long long)before + all);
        __syncthreads();
    }
    const int pieces = min(before, p.max_pieces);   // more: starts that do not ascend
    if (threadIdx.x == 0) *p.pieces = pieces;
    for (int w = threadIdx.x; w < pieces; w += PLAN_THREADS) {
        int i = 0;   // the last group whose pieces start at or before w
        for (int step = 1 << (31 - __clz(p.groups)); step; step >>= 1)
            if (i + step < p.groups && base[i + step] <= w) i += step;
        const int u = w - base[i], tiles = max(row_tiles(i), 1), rows = (starts[i + 1] - starts[i]) * p.group;
        // the tiles of one kv head's rows against one run of keys side by side, so that the keys are in L2
        Piece x;
        x.seq0 = starts[i];
        x.row0 = u % tiles * BM;
        x.rows = min(BM, rows - x.row0);
        x.kvh = u / tiles % p.hkv;
        x.split = u / tiles / p.hkv;
        x.blk0 = x.split * per;
        x.nblk = min(per, blocks_of(keys[i]) - x.blk0);
        x.keys = keys[i];
        p.piece[w] = x;
    }
    for (int b = threadIdx.x; b < p.batch; b += PLAN_THREADS) p.splits[b] = (blocks_of(in_common(p, b)) + per - 1) / per;
    pdl_wait();   // a kernel does not complete before the one ahead
}

// ----------------------------------------------------------------------------------------------------------- the prefixes
template <int HD>
struct Cfg {
    static constexpr int Q_BYTES = BM * HD, K_BYTES = BN * HD, V_BYTES = BN * HD * 2, V_HALF_BYTES = BN * 128;
    static constexpr int OFF_Q = 0;
    static constexpr int OFF_K = OFF_Q + Q_BYTES;
    static constexpr int OFF_V = OFF_K + K_STAGES * K_BYTES;
    static constexpr int OFF_RAW = OFF_V + V_STAGES * V_BYTES;
    static constexpr int OFF_BAR = OFF_RAW + RAW_STAGES * K_BYTES;
    static constexpr int SMEM = OFF_BAR + 256;
    static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "all are resident");
    // S[0], S[1] (64 columns each; P of the same block, packed fp16 pairs, over the first half of its S), O from 128 on
    static constexpr int TMEM_COLS = 256, O_COL = 128;
};

struct Params {
    const uint8_t* q;
    const int *seq_lens, *shared_lens;
    int batch, hkv, group, s_max;
    float scale_log2;
    const float *sq, *sk;
    const int* block_table;
    int max_pages, num_pages, page_size;
    FastDiv page, heads;          // heads: query heads of a kv head
    const int* pieces;
    const Piece* piece;
    float *out_o, *out_ml;        // [split][batch * q heads][HD], [..][2]
    uint32_t* status;
};

__device__ __forceinline__ Piece piece_of(const Params& p, int w) {
    const int4 a = __ldcg(reinterpret_cast<const int4*>(p.piece + w)), b = __ldcg(reinterpret_cast<const int4*>(p.piece + w) + 1);
    Piece x;
    x.seq0 = a.x; x.row0 = a.y; x.rows = a.z; x.kvh = a.w;
    x.blk0 = b.x; x.nblk = b.y; x.split = b.z; x.keys = b.w;
    return x;
}

template <int HD>
__global__ void __launch_bounds__(THREADS, CTAS)
fa_prefix_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const Params p) {
    using C = Cfg<HD>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sbase = smem_u32(smem), bars = sbase + C::OFF_BAR;
    const uint32_t bar_q = bars;                            // the piece's rows of Q are there
    const uint32_t bar_pfull = bars + 8;                    // [2] P is in tensor memory
    const uint32_t bar_kfull = bar_pfull + 16;              // [K_STAGES] K has landed
    const uint32_t bar_sfull = bar_kfull + 8 * K_STAGES;    // [K_STAGES] S is complete (K may be loaded over)
    const uint32_t bar_raw = bar_sfull + 8 * K_STAGES;      // [RAW_STAGES] codes of V have landed
    const uint32_t bar_rawfree = bar_raw + 8 * RAW_STAGES;  // [RAW_STAGES] ... and are converted
    const uint32_t bar_vfull = bar_rawfree + 8 * RAW_STAGES;   // [V_STAGES] fp16 V is there
    const uint32_t bar_pvdone = bar_vfull + 8 * V_STAGES;   // [V_STAGES] O += P V is complete (V may be converted over)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_BAR + 192);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    int* first_nan = reinterpret_cast<int*>(smem + C::OFF_BAR + 200);   // [NAN_SLOTS] of the last pieces: the first key whose V has a NaN
    const int lane = threadIdx.x & 31;
    // A scheduler has every fourth warp.  Those that convert issue as much as a softmax warp, so the second half of the CTAs, which come to the SMs of the first, has them with
    // the other two schedulers.
    const int warp_id = threadIdx.x >> 5, warp = warp_id >= SOFTMAX_WARPS && 2 * blockIdx.x >= gridDim.x ? warp_id ^ 2 : warp_id;
    if (threadIdx.x == 0) {
        mbar_init(bar_q, SOFTMAX_WARPS * 32);
        for (int s = 0; s < K_STAGES; s++) {
            mbar_init(bar_kfull + 8 * s, 1);
            mbar_init(bar_sfull + 8 * s, 1);
        }
        for (int s = 0; s < V_STAGES; s++) {
            mbar_init(bar_vfull + 8 * s, 1);
            mbar_init(bar_pvdone + 8 * s, 1);
        }
        for (int s = 0; s < RAW_STAGES; s++) {
            mbar_init(bar_raw + 8 * s, 1);
            mbar_init(bar_rawfree + 8 * s, 1);
        }
        for (int b = 0; b < 2; b++) mbar_init(bar_pfull + 8 * b, SOFTMAX_WARPS * 32);
        for (int i = 0; i < NAN_SLOTS; i++) first_nan[i] = 0x7fffffff;
        *abort_flag = sbase & 1023u ? ST_PREFIX_SMEM : 0;
        fence_mbar_init();
    }
    if (warp == MMA_WARP) {
        tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_s = *tmem_slot, tmem_o = tmem_s + C::O_COL;
    pdl_wait();
    pdl_trigger();
    const int pieces = *abort_flag ? 0 : ld_s32(p.pieces);

    if (warp == LOAD_WARP) {
        // ------------------------------------------------------------------------------------------------ loads
        const bool leader = elect_one();
        if (leader) {
            prefetch_tmap(&tmap_k);
            prefetch_tmap(&tmap_v);
        }
        int s = 0, raw = 0;
        uint32_t ph = 0, raw_ph = 0;
        bool ok = true;
        for (int w = blockIdx.x; w < pieces && ok; w += gridDim.x) {
            const Piece x = piece_of(p, w);
            int entry = 0, entries_from = 0;   // lane i: the first sequence's entry for block entries_from + i
            for (int j = 0; j < x.nblk; j++) {
                const int key0 = (x.blk0 + j) * BN;
                int row = key0, z = x.seq0 * p.hkv + x.kvh;
                if (p.block_table) {
                    if ((j & 31) == 0) {
                        entries_from = j;
                        const int key = key0 + lane * BN;
                        entry = -1;
                        if (j + lane < x.nblk) {
                            const int page = __ldcg(p.block_table + (size_t)x.seq0 * p.max_pages + p.page.div((uint32_t)key));
                            if (page >= 0 && page < p.num_pages) entry = page;
                        }
                    }
                    const int page = __shfl_sync(0xffffffffu, entry, j - entries_from);
                    row = key0 - (int)p.page.div((uint32_t)key0) * p.page_size;
                    z = page < 0 ? -1 : page * p.hkv + x.kvh;   // -1: outside the map, which arrives as zeros
                }
                ok = mbar_wait_warp(bar_sfull + 8 * s, ph ^ 1, abort_flag, ST_PREFIX_LOAD);
                if (!ok) break;
                if (leader) {
                    mbar_arrive_expect_tx(bar_kfull + 8 * s, C::K_BYTES);
                    tma_load_3d(sbase + C::OFF_K + s * C::K_BYTES, &tmap_k, bar_kfull + 8 * s, 0, row, z);
                }
                ok = mbar_wait_warp(bar_rawfree + 8 * raw, raw_ph ^ 1, abort_flag, ST_PREFIX_LOAD);
                if (!ok) break;
                if (leader) {
                    mbar_arrive_expect_tx(bar_raw + 8 * raw, C::K_BYTES);
                    tma_load_3d(sbase + C::OFF_RAW + raw * C::K_BYTES, &tmap_v, bar_raw + 8 * raw, 0, row, z);
                }
                __syncwarp();
                if (++s == K_STAGES) { s = 0; ph ^= 1; }
                if (++raw == RAW_STAGES) { raw = 0; raw_ph ^= 1; }
            }
        }
    } else if (warp >= CONVERT_WARP) {
        // -------------------------------------------------------------------------------------- V: codes -> fp16
        // two warps in turn: one takes as long for a block as the softmax warps do
        const bool leader = elect_one();
        const uint32_t mine = warp - CONVERT_WARP;
        uint32_t block = 0, nth = 0;   // blocks and pieces before this one
        bool ok = true;
        for (int w = blockIdx.x; w < pieces && ok; w += gridDim.x, nth++) {
            const Piece x = piece_of(p, w);
            for (int j = 0; j < x.nblk; j++, block++) {
                if (block % CONVERTERS != mine) continue;
                const uint32_t raw = block % RAW_STAGES, s = block % V_STAGES;
                ok = mbar_wait_warp(bar_raw + 8 * raw, block / RAW_STAGES & 1, abort_flag, ST_PREFIX_CONVERT) &&
                     mbar_wait_warp(bar_pvdone + 8 * s, (block / V_STAGES & 1) ^ 1, abort_flag, ST_PREFIX_CONVERT);
                if (!ok) break;
                // The slot of the piece after next is cleared: neither warp is that far (its P V would be two ahead of one that needs this block), and whoever reads it for six
                // pieces back has done so (this block has waited for the P V two blocks back).
                if (j == 0 && leader) first_nan[(nth + 2) % NAN_SLOTS] = 0x7fffffff;
                const uint32_t from = sbase + C::OFF_RAW + raw * C::K_BYTES, to = sbase + C::OFF_V + s * C::V_BYTES;
                const int key0 = (x.blk0 + j) * BN, valid = x.keys - key0;
                if (valid < BN) {   // what lies behind the common keys may be anything: no weight of zero may meet it
                    for (int i = lane; i < (BN - valid) * (HD / 16); i += 32)
                        asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(from + valid * HD + 16 * i), "r"(0) : "memory");
                    __syncwarp();
                }
                if (convert_v<HD, true>(from, to)) {   // rare: which key is the first
                    for (int key = 0; key < BN; key++)
                        for (int d = 0; d < HD; d += 4) {
                            uint32_t c;
                            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(c) : "r"(from + key * HD + d) : "memory");
                            if (((c & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) {
                                atomicMin(first_nan + nth % NAN_SLOTS, key0 + key);
                                key = BN;
                                break;
                            }
                        }
                }
                __syncwarp();
                fence_proxy_async_smem();
                __syncwarp();
                if (leader) {
                    mbar_arrive(bar_vfull + 8 * s);
                    mbar_arrive(bar_rawfree + 8 * raw);
                }
                __syncwarp();
            }
        }
    } else if (warp == MMA_WARP) {
        // --------------------------------------------------------------------------------------------- products
        const bool leader = elect_one();
        float sign = p.scale_log2;   // of a negative scale the scores come with the sign that their maximum is taken with
        if (p.sq) sign *= ld_f32(p.sq);
        if (p.sk) sign *= ld_f32(p.sk);
        const uint32_t idesc_qk = make_idesc_e4m3_f32(BM, BN, 0, 0) | (sign < 0.f ? IDESC_NEGATE_A : 0u);
        constexpr uint32_t idesc_pv = make_idesc_f16_f32(BM, HD, 0, 1);   // P from tensor memory, V is MN-major
        auto desc = [&](uint32_t addr) { return HD == 128 ? kmajor_desc_sw128(addr) : kmajor_desc_sw64(addr); };
        int ks = 0, vs = 0;
        uint32_t kph = 0, vph = 0, kb = 0, vb = 0, pph = 0, qph = 0;
        bool ok = true;
        auto issue_qk = [&]() {   // S[kb] = Q K^T of the next block
            ok = mbar_wait_warp(bar_kfull + 8 * ks, kph, abort_flag, ST_PREFIX_MMA);
            if (!ok) return;
            tc_fence_after();
            const uint64_t qd = desc(sbase + C::OFF_Q), kd = desc(sbase + C::OFF_K + ks * C::K_BYTES);
            if (leader) {
#pragma unroll
                for (int k = 0; k < HD / 32; k++) mma_f8f6f4_ss(tmem_s + kb * BN, qd + 2 * k, kd + 2 * k, idesc_qk, k != 0);
                mma_commit(bar_sfull + 8 * ks);
            }
            __syncwarp();
            kb ^= 1;
            if (++ks == K_STAGES) { ks = 0; kph ^= 1; }
        };
        for (int w = blockIdx.x; w < pieces && ok; w += gridDim.x) {
            const int nblk = piece_of(p, w).nblk;
            ok = mbar_wait_warp(bar_q, qph, abort_flag, ST_PREFIX_MMA);
            qph ^= 1;
            // two blocks' scores ahead of the P V
            for (int i = 0; i < 2 && i < nblk && ok; i++) issue_qk();
            for (int j = 0; j < nblk && ok; j++) {
                const uint32_t b = vb;
                ok = mbar_wait_warp(bar_vfull + 8 * vs, vph, abort_flag, ST_PREFIX_MMA) && mbar_wait_warp(bar_pfull + 8 * b, (pph >> b) & 1, abort_flag, ST_PREFIX_MMA);
                if (!ok) break;
                pph ^= 1u << b;
                vb ^= 1;
                tc_fence_after();
                const uint32_t vaddr = sbase + C::OFF_V + vs * C::V_BYTES;
                if (leader) {
#pragma unroll
                    for (int k = 0; k < BN / 16; k++) {   // 16 keys: 8 columns of P, 16 rows of V
                        const uint64_t vd = mnmajor_desc_sw128(vaddr + k * 16 * 128, C::V_HALF_BYTES);
                        mma_f16_ts(tmem_o, tmem_s + b * BN + 8 * k, vd, idesc_pv, (j | k) != 0);
                    }
                    mma_commit(bar_pvdone + 8 * vs);
                }
                __syncwarp();
                if (++vs == V_STAGES) { vs = 0; vph ^= 1; }
                // behind this P V on the same in-order pipe: P has been read before S lands on it
                if (j + 2 < nblk) issue_qk();
            }
        }
    } else {
        // ------------------------------------------------------------------------------------- a row to a thread
        const int r = threadIdx.x;
        const uint32_t lane_off = uint32_t(warp * 32) << 16;
        float scale_log2 = p.scale_log2;
        if (p.sq) scale_log2 *= ld_f32(p.sq);
        if (p.sk) scale_log2 *= ld_f32(p.sk);
        float ascale = fabsf(scale_log2);
        if (ascale == 0.f) ascale = 1e-30f;   // keeps -inf * scale = -inf for masked keys
        uint32_t block = 0, nth = 0;     // blocks and pieces before this one
        auto wait_pv = [&](uint32_t of) { return mbar_wait_warp(bar_pvdone + 8 * (of % V_STAGES), of / V_STAGES & 1, abort_flag, ST_PREFIX_SOFTMAX); };
        bool ok = true;
        for (int w = blockIdx.x; w < pieces && ok; w += gridDim.x, nth++) {
            const Piece x = piece_of(p, w);
            const bool idle = warp * 32 >= x.rows;   // no row of this warp is any
            // ---- this row's codes, at the swizzle's places; the last Q K^T of the piece before is complete
            uint32_t row = 0;
            int lim = 0x7fffffff;   // keys of the prefix that it sees; a row that is none sees all, of a query of zeros
            const uint32_t q_at = sbase + C::OFF_Q + r * HD;
            if (r < x.rows) {
                uint32_t s, h;
                p.heads.divmod((uint32_t)(x.row0 + r), s, h);
                const int b = x.seq0 + (int)s;
                lim = min(min(max(__ldcg(p.seq_lens + b), 0), p.s_max), max(__ldcg(p.shared_lens + b), 0));
                row = ((uint32_t)b * p.hkv + x.kvh) * p.group + h;
            }
            if (!idle) {
                uint4 c[HD / 16];
#pragma unroll
                for (int i = 0; i < HD / 16; i++) c[i] = r < x.rows ? ld128(p.q + (size_t)row * HD + 16 * i) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                for (int i = 0; i < HD / 16; i++)
                    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(q_at + ((HD == 128 ? i ^ (r & 7) : i ^ ((r >> 1) & 3)) << 4)), "r"(c[i].x), "r"(c[i].y), "r"(c[i].z), "r"(c[i].w)
                                 : "memory");
            }
            const int all_see = __reduce_min_sync(0xffffffffu, lim);   // keys that all rows of this warp see
            fence_proxy_async_smem();
            mbar_arrive(bar_q);
            float m_ref = -INFINITY, nmsub = 0.f, l = 0.f;
            for (int j = 0; j < x.nblk; j++, block++) {
                const uint32_t buf = block & 1, sa = tmem_s + lane_off + buf * BN;
                ok = mbar_wait_warp(bar_sfull + 8 * (block % K_STAGES), block / K_STAGES & 1, abort_flag, ST_PREFIX_SOFTMAX);
                if (!ok) break;
                tc_fence_after();
                if (!idle) {
                    uint32_t sreg[BN];
#pragma unroll
                    for (int c = 0; c < BN / 32; c++) tmem_ld_32x32b_x32(sa + c * 32, sreg + c * 32);
                    tmem_ld_wait();
                    const int key0 = (x.blk0 + j) * BN;
                    if (all_see - key0 < BN) {
                        const int seen = lim - key0;   // keys of the block that this row sees
                        if (__any_sync(0xffffffffu, seen > 0 && seen < BN)) {   // an edge
#pragma unroll
                            for (int c = 0; c < BN; c++)
                                if (c >= seen) sreg[c] = 0xff800000u;
                        } else {
                            const bool blind = seen <= 0;
#pragma unroll
                            for (int c = 0; c < BN; c++)
                                if (blind) sreg[c] = 0xff800000u;
                        }
                    }
                    float l0 = 0.f, l1 = 0.f, l2 = 0.f, l3 = 0.f;   // of this block
                    float mxa[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) mxa[i] = fmaxf(__uint_as_float(sreg[2 * i]), __uint_as_float(sreg[2 * i + 1]));
#pragma unroll
                    for (int c = 8; c < BN; c += 8)
#pragma unroll
                        for (int i = 0; i < 4; i++) mxa[i] = max3(mxa[i], __uint_as_float(sreg[c + 2 * i]), __uint_as_float(sreg[c + 2 * i + 1]));
                    const float mx = fmaxf(fmaxf(mxa[0], mxa[1]), fmaxf(mxa[2], mxa[3])) * ascale;
                    if (__any_sync(0xffffffffu, mx > m_ref + TAU)) {   // rare once a few blocks are in
                        const bool bump = mx > m_ref + TAU;
                        const float m_new = bump ? mx : m_ref;
                        if (j > 0) {   // O is final only once the P V before is
                            ok = wait_pv(block - 1);
                            if (!ok) break;
                            tc_fence_after();
                            const float f = bump ? ex2(m_ref - m_new) : 1.0f;   // m_ref = -inf -> 0
                            l *= f;
#pragma unroll
                            for (int c = 0; c < HD / 8; c++) {   // (eight columns: of more, the scores would not stay in registers)
                                uint32_t o[8];
                                tmem_ld_32x32b_x8(tmem_o + lane_off + c * 8, o);
                                tmem_ld_wait();
#pragma unroll
                                for (int i = 0; i < 8; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                                tmem_st_32x32b_x8(tmem_o + lane_off + c * 8, o);
                            }
                        }
                        m_ref = m_new;
                        nmsub = m_ref == -INFINITY ? 0.f : POFF - m_ref;
                    }
#pragma unroll
                    for (int g = 0; g < BN / 32; g++) {   // 32 keys -> 16 columns
                        uint32_t pw[16];
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            float x0, x1;
                            ffma2(x0, x1, __uint_as_float(sreg[g * 32 + 2 * i]), __uint_as_float(sreg[g * 32 + 2 * i + 1]), ascale, ascale, nmsub, nmsub);
                            const float p0 = ex2(x0), p1 = ex2(x1);
                            if (i & 1) fadd2(l2, l3, p0, p1); else fadd2(l0, l1, p0, p1);
                            pw[i] = pack_half2(p0, p1);
                        }
                        tmem_st_32x32b_x16(sa + g * 16, pw);
                    }
                    l += (l0 + l1) + (l2 + l3);
                    tmem_st_wait();
                }
                tc_fence_before();
                mbar_arrive(bar_pfull + 8 * buf);
            }
            if (!ok) break;
            // ---- the piece's state of this row.  Every warp waits, also one without rows: the next piece's Q and P go over what the products read
            ok = wait_pv(block - 1);
            if (!ok) break;
            tc_fence_after();
            if (!idle) {
                // V was 2^-8 of itself; where a value that the row sees is a NaN, all columns become one (the weights, and with them the LSE, are what they are)
                const float v_scale = lim > *(volatile int*)(first_nan + nth % NAN_SLOTS) ? NAN : 256.f;
                const size_t at = (size_t)x.split * p.batch * p.hkv * p.group + row;
#pragma unroll
                for (int c = 0; c < HD / 64; c++) {
                    uint32_t o[64];
                    tmem_ld_32x32b_x32(tmem_o + lane_off + c * 64, o);
                    tmem_ld_32x32b_x32(tmem_o + lane_off + c * 64 + 32, o + 32);
                    tmem_ld_wait();
                    if (r < x.rows) {
                        // columns come in the order 0, 2, 1, 3 of four
                        auto f = [&](int i) { return __uint_as_float(o[(i & ~3) | (i & 1) << 1 | (i >> 1 & 1)]) * v_scale; };
#pragma unroll
                        for (int i = 0; i < 64; i += 8)
                            asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p.out_o + at * HD + c * 64 + i), "f"(f(i)), "f"(f(i + 1)), "f"(f(i + 2)), "f"(f(i + 3)),
                                         "f"(f(i + 4)), "f"(f(i + 5)), "f"(f(i + 6)), "f"(f(i + 7)) : "memory");
                    }
                }
                if (r < x.rows) *reinterpret_cast<float2*>(p.out_ml + 2 * at) = make_float2(m_ref - POFF, l);
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    const uint32_t code = *abort_flag;
    if (code != 0) {
        if (threadIdx.x == 0) atomicCAS(p.status, 0u, code);
        for (int i = 0; i < 200; i++) __nanosleep(1000);   // let copies already in flight land
        __syncthreads();
    }
    if (warp == MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem_s, C::TMEM_COLS);
    }
}

// A row's state of the keys that its sequence has to itself and those of the pieces, added up.  D / 4 threads to a row: four times as many, each with a quarter of the pieces,
// take more CTAs (400 sequences behind 1000 keys 41 -> 58 us; 32 behind 12000 34.3 -> 33.1).
struct SumParams {
    const float *own_o, *own_ml, *out_o, *out_ml;
    const int* splits;
    __half* o;
    float* lse;
    int rows;            // batch * q heads
    FastDiv q_heads;
    float v_descale;
    const float* sv;
};
constexpr int SUM_THREADS = 128;
template <int D>
__global__ void __launch_bounds__(SUM_THREADS) prefix_sum_kernel(const SumParams p) {
    constexpr int ROWS = SUM_THREADS / (D / 4);   // of a CTA
    const int row = blockIdx.x * ROWS + threadIdx.x / (D / 4), col = threadIdx.x % (D / 4) * 4;
    pdl_wait();
    pdl_trigger();
    if (row >= p.rows) return;
    const int n = __ldcg(p.splits + p.q_heads.div((uint32_t)row));
    const float vds = p.sv ? p.v_descale * ld_f32(p.sv) : p.v_descale;
    State s;
    s.add_all<D>(p.own_ml, p.own_o, 1, col, [&](int) { return (size_t)row; });
    s.add_all<D>(p.out_ml, p.out_o, n, col, [&](int i) { return (size_t)i * p.rows + row; });
    store_output<D>(p.o, p.lse, row, col, s, vds);
}

// The workspace: the plan, the states, then what the stream kernel keeps.
struct Layout {
    int max_splits, resident, max_pieces;
    size_t pieces, piece, splits, ml, o, own_ml, own_o, stream, bytes;
};
size_t up(size_t x) { return (x + 255) & ~(size_t)255; }

struct Call {
    StreamArgs a;
    const int* starts;
    int groups;
    Layout x;
};

Layout layout_of(const StreamArgs& a, int groups) {
    Layout x;
    x.resident = CTAS * sms_of_current_device();
    const long long rows = (long long)a.batch * a.q_heads, group = a.q_heads / a.kv_heads;
    const long long tiles = (a.batch * group + BM - 1) / BM * a.kv_heads;   // of one group of all
    const long long splits = (x.resident + tiles - 1) / tiles;
    x.max_splits = (int)(splits > MAX_SPLITS ? MAX_SPLITS : splits);
    const long long pieces = (a.batch * group / BM + groups) * a.kv_heads * x.max_splits;
    x.max_pieces = (int)(pieces > 0x3ffffff ? 0 : pieces);   // 0: more than can be planned
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at = up(at + bytes);
        return here;
    };
    x.pieces = take(4);
    x.splits = take((size_t)a.batch * 4);
    x.piece = take((size_t)x.max_pieces * sizeof(Piece));
    x.ml = take((size_t)x.max_splits * rows * 8);
    x.o = take((size_t)x.max_splits * rows * a.hd * 4);
    x.own_ml = take((size_t)rows * 8);
    x.own_o = take((size_t)rows * a.hd * 4);
    x.stream = take(stream_workspace_bytes(a));
    x.bytes = at;
    return x;
}

template <int HD>
cudaError_t run(const StreamArgs& a, const Params& p, const SumParams& sum, int grid) {
    using C = Cfg<HD>;
    cudaError_t e = cudaFuncSetAttribute(fa_prefix_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    const uint64_t outer = (uint64_t)(a.block_table ? a.num_pages : a.batch) * a.kv_heads, rows = (uint64_t)(a.block_table ? a.page_size : a.s_max);
    CUtensorMap k, v;
    if (!make_tmap_u8_3d(&k, a.k_cache, outer, rows, HD, BN, HD, HD == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B) ||
        !make_tmap_u8_3d(&v, a.v_cache, outer, rows, HD, BN, HD, HD == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE))
        return cudaErrorInvalidValue;
    e = launch_pdl(fa_prefix_kernel<HD>, dim3((unsigned)grid), dim3(THREADS), C::SMEM, a.stream, k, v, p);
    if (e != cudaSuccess) return e;
    const long long ctas = ((long long)sum.rows * (HD / 4) + SUM_THREADS - 1) / SUM_THREADS;
    return launch_pdl(prefix_sum_kernel<HD>, dim3((unsigned)ctas), dim3(SUM_THREADS), 0, a.stream, sum);
}

cudaError_t launch_shared(const void* args, const CallScratch& scratch) {
    const Call& c = *static_cast<const Call*>(args);
    const Layout& x = c.x;
    StreamArgs a = c.a;
    uint8_t* ws = static_cast<uint8_t*>(scratch.workspace);
    a.own_o = reinterpret_cast<float*>(ws + x.own_o);
    a.own_ml = reinterpret_cast<float*>(ws + x.own_ml);
    a.workspace = ws + x.stream;
    a.arrivals = scratch.zeros;
    cudaError_t e = launch_stream(a);
    if (e != cudaSuccess) return e;
    PlanParams plan;
    plan.seq_lens = a.seq_lens; plan.shared_lens = a.shared_lens; plan.starts = c.starts;
    plan.batch = a.batch; plan.groups = c.groups; plan.group = a.q_heads / a.kv_heads; plan.hkv = a.kv_heads; plan.s_max = a.s_max;
    plan.max_splits = x.max_splits; plan.max_pieces = x.max_pieces; plan.resident = x.resident;
    plan.pieces = reinterpret_cast<int*>(ws + x.pieces);
    plan.piece = reinterpret_cast<Piece*>(ws + x.piece);
    plan.splits = reinterpret_cast<int*>(ws + x.splits);
    e = launch_pdl(prefix_plan_kernel, dim3(1), dim3(PLAN_THREADS), (3 * (size_t)c.groups + 1) * 4, a.stream, plan);
    if (e != cudaSuccess) return e;
    Params p;
    p.q = static_cast<const uint8_t*>(a.q);
    p.seq_lens = a.seq_lens; p.shared_lens = a.shared_lens;
    p.batch = a.batch; p.hkv = a.kv_heads; p.group = a.q_heads / a.kv_heads; p.s_max = a.s_max;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.sq = a.scale_q_dev; p.sk = a.scale_k_dev;
    p.block_table = a.block_table;
    p.max_pages = a.max_pages; p.num_pages = a.num_pages; p.page_size = a.page_size;
    p.page = FastDiv(a.block_table ? (uint32_t)a.page_size : 1u);
    p.heads = FastDiv((uint32_t)p.group);
    p.pieces = plan.pieces;
    p.piece = plan.piece;
    p.out_o = reinterpret_cast<float*>(ws + x.o);
    p.out_ml = reinterpret_cast<float*>(ws + x.ml);
    p.status = status_word();
    if (!p.status) return cudaErrorInvalidSymbol;
    SumParams sum;
    sum.own_o = a.own_o; sum.own_ml = a.own_ml; sum.out_o = p.out_o; sum.out_ml = p.out_ml;
    sum.splits = plan.splits;
    sum.o = static_cast<__half*>(a.o);
    sum.lse = a.lse;
    sum.rows = a.batch * a.q_heads;
    sum.q_heads = FastDiv((uint32_t)a.q_heads);
    sum.v_descale = a.v_descale;
    sum.sv = a.scale_v_dev;
    const int grid = x.max_pieces < x.resident ? x.max_pieces : x.resident;
    return a.hd == 128 ? run<128>(a, p, sum, grid) : run<64>(a, p, sum, grid);
}

}  // namespace

}  // namespace fa_sm100

extern "C" fa_status_t fa_decode_shared(fa_ctx_t* ctx, const fa_decode_args_t* g, const int* shared_lens, const int* group_starts, int groups) {
    using namespace fa_sm100;
    const char* who = "fa_decode_shared";
    if (!ctx) return FA_ERR_INVALID_ARG;
    int s_max = 0;
    const fa_status_t ok = check_stream(ctx, who, g, s_max);
    if (ok != FA_OK) return ok;
    if (!g->seq_lens || !shared_lens || !group_starts || groups <= 0) return refuse(ctx, who, FA_ERR_INVALID_ARG, "seq_lens, shared_lens and group_starts are needed, and groups > 0");
    if ((reinterpret_cast<uintptr_t>(shared_lens) | reinterpret_cast<uintptr_t>(group_starts)) & 3) return refuse(ctx, who, FA_ERR_INVALID_ARG, "shared_lens and group_starts must be 4-byte aligned");
    if (groups > g->batch) return refuse(ctx, who, FA_ERR_INVALID_ARG, "there are more groups than sequences");
    if (groups > MAX_GROUPS) return refuse(ctx, who, FA_ERR_UNSUPPORTED_SHAPE, "at most 2048 groups");
    Call c;
    c.a = stream_args(*g, s_max);
    if ((double)(g->batch - groups) * s_max * g->kv_heads * g->head_dim * 2 <= own_bytes(g->head_dim)) return launch_stream_call(ctx, who, c.a);
    c.a.shared_lens = shared_lens;
    c.starts = group_starts;
    c.groups = groups;
    c.x = layout_of(c.a, groups);
    if (c.x.max_pieces == 0) return refuse(ctx, who, FA_ERR_UNSUPPORTED_SHAPE, "more groups and heads than can be planned");
    return call_with_scratch(ctx, who, c.a.stream, c.x.bytes, stream_arrivals(c.a), launch_shared, &c);
}
