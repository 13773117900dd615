// fa_convert_v.cuh — V for a product on fp16: e4m3 codes -> fp16, exact, in registers and for a tile in shared memory.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace fa_sm100 {

constexpr int V_KEYS = 64;   // of a tile

__device__ __forceinline__ void e4m3x16_to_f16(const uint4 c, uint4& lo, uint4& hi) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    uint32_t h[8];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, u;\n\t}" : "=r"(h[2 * k]), "=r"(h[2 * k + 1]) : "r"(w[k]));
    }
    lo = make_uint4(h[0], h[1], h[2], h[3]);
    hi = make_uint4(h[4], h[5], h[6], h[7]);
}
// The same by integer operations, which leave the unit that converts (and takes exponentials) alone: a code's bits seven to the left are 2^-8 of its value as
// fp16, a subnormal one's too.  Of four codes the first and third come first, then the second and fourth.  A NaN becomes a number: nan collects, byte by byte, a
// top bit for each (it is the only code whose low seven bits are all ones).
__device__ __forceinline__ void e4m3x16_to_f16_bits(const uint4 c, uint4& lo, uint4& hi, uint32_t& nan) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    uint32_t h[8];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t up = w[k] << 8;
        h[2 * k] = (up & 0x80008000u) | ((up >> 1) & 0x3f803f80u);
        h[2 * k + 1] = (w[k] & 0x80008000u) | ((w[k] >> 1) & 0x3f803f80u);
        nan |= (w[k] & 0x7f7f7f7fu) + 0x01010101u;
    }
    lo = make_uint4(h[0], h[1], h[2], h[3]);
    hi = make_uint4(h[4], h[5], h[6], h[7]);
}
// One 64-key tile of V in shared memory: codes -> fp16 in the order of a TMA load with 128-byte swizzle, one 64-column slab of
// d after the other.  By one warp, which takes 16 codes of a lane at a time; eight neighbouring lanes, whose 16-byte accesses
// share a wavefront, meet eight different bank groups on both sides.
//  D = 128 (codes swizzled too): they take four neighbouring pieces of one slab of two keys k and k ^ 5 — bit 2 of the key puts the
//   loads in different halves of the 128 bytes, bit 0 the stores on chunks of different parity;
//  D = 64 (codes as they lie in global memory): the four pieces of two neighbouring keys, 128 bytes in a row.
// In rounds of eight steps: code that is not there is not fetched (see the loops of the softmax warps).
// BITS: by integer operations, with their order, scale and numbers for NaNs; returns whether any of this lane's codes is one.
template <int HD, bool BITS = false>
__device__ __forceinline__ bool convert_v(uint32_t raw, uint32_t dst) {
    constexpr int STEPS = V_KEYS * HD / 512, BATCH = 8;   // steps of the warp, loads in flight
    const int lane = threadIdx.x & 31;
    const int slab = HD == 128 ? (lane >> 3) & 1 : 0;
    const int key = HD == 128 ? (lane >> 4) ^ ((lane & 4) ? 5 : 0) : lane >> 2;   // of step 0, below 8
    const int chunk = ((lane & 3) * 2) ^ key;
    // D = 128: a step takes four keys, {0, 5, 1, 4} and then {2, 7, 3, 6} of eight: key + 2 is key ^ 2.  D = 64: eight
    constexpr int TURN = HD == 128 ? 2 : 1;           // steps per eight keys
    uint32_t src[TURN], lo_at[TURN], hi_at[TURN];
#pragma unroll
    for (int t = 0; t < TURN; t++) {
        const int row = (key ^ (2 * t)) * 128;
        src[t] = raw + (HD == 128 ? row + (((slab * 4 + (lane & 3)) ^ key ^ (2 * t)) << 4) : lane * 16);
        lo_at[t] = dst + slab * (V_KEYS * 128) + row + ((chunk ^ (2 * t)) << 4);
        hi_at[t] = dst + slab * (V_KEYS * 128) + row + ((chunk ^ (2 * t) ^ 1) << 4);
    }
    uint32_t nan = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < STEPS; i0 += BATCH) {
        uint4 v[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; i++)
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[i].x), "=r"(v[i].y), "=r"(v[i].z), "=r"(v[i].w)
                         : "r"(src[i % TURN] + (i0 + i) / TURN * (8 * HD)) : "memory");
#pragma unroll
        for (int i = 0; i < BATCH; i++) {
            uint4 lo, hi;
            if (BITS) e4m3x16_to_f16_bits(v[i], lo, hi, nan);
            else e4m3x16_to_f16(v[i], lo, hi);
            const int at = (i0 + i) / TURN * 1024;
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(lo_at[i % TURN] + at), "r"(lo.x), "r"(lo.y), "r"(lo.z), "r"(lo.w) : "memory");
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(hi_at[i % TURN] + at), "r"(hi.x), "r"(hi.y), "r"(hi.z), "r"(hi.w) : "memory");
        }
    }
    return (nan & 0x80808080u) != 0;
}

}  // namespace fa_sm100
